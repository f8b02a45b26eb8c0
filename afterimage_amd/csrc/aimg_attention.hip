// Attention of packed prompts, and of drafted tokens over a paged cache (gfx950).
//
// For a query row q with the keys j it sees,
//   s_j = c q.k_j,  m = max_j s_j,  l = sum_j 2^(s_j - m),  o = sum_j 2^(s_j - m) v_j / l,
// with c = scale * log2(e), in one pass over the keys: m, l and o are kept in
// fp32 and o and l are multiplied by 2^(m_old - m_new) where m rises. A row
// that sees no key gives zeros.
//
// Products. Keys are the rows and queries the columns of S^T = K Q^T
// (v_mfma_f32_32x32x16): a lane then holds 16 of 32 scores of ONE query, so
// the maximum and the sum are lane sums and one exchange of the wave's halves,
// and the probabilities are already laid out as the second operand of
// O^T = V^T P^T. The key order inside a step of 16 is the one S^T leaves them
// in (the sum over keys does not depend on it); V^T comes out of LDS through
// the transposing read (ds_read_b64_tr_b16) in that order. No probability
// passes through LDS or another lane.
//
// Rounding. q, k, v enter the products as they are; scores, m, l and o are
// fp32. Probabilities are rounded once to the inputs' type for the second
// product (l sums them unrounded), and the result once at the end.
//
// Rows of K and V go to LDS with asynchronous 16-byte loads, two tiles in
// turn; their 16-byte pieces are permuted within a row (by the row's index) so
// that neither read meets a bank twice.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>
#include <type_traits>

#include "afterimage_decode.h"
#include "aimg_internal.h"

namespace aimg {
namespace {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) int i32x2;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

struct Bf16 {
    static constexpr uint32_t kInf = 0x7F80u, kOne = 0x3F80u;
    static __device__ f32x16 mfma(s16x8 a, s16x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ uint32_t pack(float a, float b) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
    }
    // Eight e4m3 elements times a power of two, exact.
    static __device__ s16x8 from8(uint32_t a, uint32_t b, float scale) {
        auto two = [](auto x) { return __builtin_bit_cast(uint32_t, x); };
        return __builtin_bit_cast(s16x8, (u32x4{two(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, false)),
                                                two(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, true)),
                                                two(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, false)),
                                                two(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, true))}));
    }
};

struct Fp16 {
    static constexpr uint32_t kInf = 0x7C00u, kOne = 0x3C00u;
    static __device__ f32x16 mfma(s16x8 a, s16x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ uint32_t pack(float a, float b) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), f16x2));
    }
    static __device__ s16x8 from8(uint32_t a, uint32_t b, float scale) {
        auto two = [](auto x) { return __builtin_bit_cast(uint32_t, x); };
        return __builtin_bit_cast(s16x8, (u32x4{two(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, scale, false)),
                                                two(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, scale, true)),
                                                two(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, scale, false)),
                                                two(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, scale, true))}));
    }
};

// m need not be the maximum itself: any number near enough keeps 2^(s - m) in
// range, and the quotient o / l is the same. It is set at a row's first visible
// tile and then left alone while a lane's sum of 32 (or 16) probabilities
// stays below kMostSum, so that each is far inside the range of both types; a
// tile then needs no maximum and o and l no multiplication. Where the sum is
// more, some probability is over 2^9 and the maximum is raised if it grew by
// more than 2^kRise.
constexpr float kMostSum = 16384.0f;
constexpr float kRise = 8.0f;
constexpr float kLog2E = 1.44269504088896340736f;
constexpr int kMaxDim = 256;
constexpr int64_t kMaxRowStride = 1 << 24;  // 64 rows stay within 32-bit byte offsets

// Rows of a tile in LDS: row r of kBytes bytes, its 16-byte piece x at place
// x ^ key_place(r) or x ^ value_place(r).
// Keys are read 16 bytes a lane, one row a lane: 16 rows (8 of 128 bytes) at
// one x cover all banks. Values are read by four rows and two neighbouring
// pieces at a time (four pieces for two groups of lanes): {0,6,10,12} takes
// pairs to four places of 32 bytes mod 128 and fours to four of 64 mod 256.
template <int DP>
struct Rows {
    static constexpr int kBytes = DP * 2;
    static constexpr int kPieces = DP / 8;
    static constexpr int kPerLoad = 64 / kPieces;  // rows of one load of 64 lanes
    static __device__ int key_place(int r) { return r & (DP == 64 ? 7 : 15); }
    static __device__ int value_place(int r) {
        r &= 3;
        return DP == 64 ? 2 * r : 4 * r ^ 2 * ((r ^ r >> 1) & 1);
    }
};

// Rows of a tile of 8-bit elements, pieces of 16. Keys: 16 rows at one x cover
// all banks once (rows of 64 bytes take four places for each four rows). Values
// are read by eight rows {0..3, 8..11} (+ 4) and two neighbouring pieces at a time.
template <int DP>
struct Rows8 {
    static constexpr int kBytes = DP;
    static constexpr int kPieces = DP / 16;
    static constexpr int kPerLoad = 64 / kPieces;
    static __device__ int key_place(int r) { return DP == 64 ? r >> 2 & 3 : DP == 128 ? r >> 1 & 7 : r & 15; }
    static __device__ int value_place(int r) { return DP == 64 ? r >> 2 & 2 : DP == 128 ? (r & 2) | (r >> 1 & 4) : 2 * (r & 3) | (r & 8); }
};

constexpr int kBlock = 16;  // positions that share a scale in a cache of 8 bits

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The larger of a lane's value and that of the same query in the wave's other half.
__device__ __forceinline__ float max_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ float add_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

typedef __attribute__((address_space(3))) char lds_char;

__device__ __forceinline__ void load_to_lds(const void* from, lds_char* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

__device__ __forceinline__ void load4_to_lds(const void* from, lds_char* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)to, 4, 0, 0);
}

// Keys narrower than DP elements: the pieces past a row's last, which hold a
// copy of it, become zeros in rows row0 .. row0 + kRows - 1 of the tile, that
// the wave itself has loaded. (An infinite element of the copy would meet the
// query's zeros there and make the score NaN. Lanes that sit those loads out
// instead, over places cleared once: 32 trees of dim 96 over 2000-8000
// positions 130 us.)
template <typename R, int kRows>
__device__ __forceinline__ void clear_past(int pieces, lds_char* keys, int row0, int lane) {
    asm volatile("" : "+v"(lane));  // its addresses are not worth registers in the loop over tiles
    const int r = row0 + lane % kRows;
    for (int x = pieces + lane / kRows; x < R::kPieces; x += 64 / kRows)
        *reinterpret_cast<__attribute__((address_space(3))) u32x4*>(keys + r * R::kBytes + ((x ^ R::key_place(r)) << 4)) = u32x4{0};
}

// x where bit `at` of bits is set, -inf otherwise: two instructions, and no lane mask in scalar registers.
__device__ __forceinline__ float seen_or(uint32_t bits, int at, float x) {
    const uint32_t all = static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(bits), at, 1));
    return __uint_as_float((__float_as_uint(x) & all) | (0xFF800000u & ~all));
}

// Waits until at most kLeft of the wave's vector memory loads are in flight.
template <int kLeft>
__device__ __forceinline__ void wait_loads() {
    __builtin_amdgcn_s_waitcnt((kLeft & 15) | (kLeft >> 4) << 14 | 0x0F70);
    asm volatile("" ::: "memory");
}

// One wave's softmax state and output of QT tiles of 32 queries.
// Keys and values of 8 bits become bf16 times their scales, which is exact;
// for queries in fp16, keys become fp16 as they are, exact too, and scores are
// multiplied by their keys' scales. Values are bf16 for either (their range may
// pass fp16's), and fp16 queries' probabilities the sum of two bf16 numbers,
// which 16 bits of them are in.
// A lane reads 16 elements of such a key at a time, which serve two steps of the
// first product (the queries are laid out likewise).
template <typename T, int DP, int QT, bool k8 = false>
struct State {
    static constexpr bool kScaled = k8 && std::is_same_v<T, Fp16>;
    typedef std::conditional_t<k8, Bf16, T> P;  // of the second product
    typedef std::conditional_t<k8, Rows8<DP>, Rows<DP>> R;
    struct Scales {};
    struct Scales8 {
        const __attribute__((address_space(3))) float* at;  // a tile's keys' scales, then its values'
        int blocks;
    };
    typedef std::conditional_t<k8, Scales8, Scales> TileScales;
    static constexpr int kSteps = DP / 16;   // steps of the first product
    static constexpr int kBlocks = DP / 32;  // blocks of output columns
    s16x8 q[QT][kSteps];
    f32x16 o[QT][kBlocks];
    float m[QT], l[QT];

    __device__ void clear() {
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            m[t] = -INFINITY;
            l[t] = 0.0f;
#pragma unroll
            for (int d = 0; d < kBlocks; ++d) o[t][d] = f32x16{0};
        }
    }

    // A lane's query row (dim elements, the rest zero), in the layout of the second operand.
    __device__ void load_query(int t, const uint16_t* row, int dim, int half) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            const int x = k8 ? 32 * (k / 2) + 16 * half + 8 * (k % 2) : 8 * (2 * k + half);
            const s16x8 v = *reinterpret_cast<const s16x8*>(row + (x < dim ? x : 0));
            q[t][k] = x < dim ? v : s16x8{0};
        }
    }

    // The next 32 * NSUB keys, their rows at `keys` and `values` in LDS.
    // kMasked: allow[t][u] has bit r set where the lane's query of tile t sees
    // key 32 u + r; every key is seen otherwise.
    template <int NSUB, bool kMasked>
    __device__ __forceinline__ void step(const lds_char* keys, const lds_char* values, float c, int lane,
                                         const uint32_t (&allow)[QT][NSUB], const TileScales& scales = {}) {
        const int half = lane >> 5;
        f32x16 s[QT][NSUB];
#pragma unroll
        for (int u = 0; u < NSUB; ++u) {
            const int r = lane & 31;
            const lds_char* const row = keys + (32 * u + r) * R::kBytes;
            if constexpr (k8) {
                const float scale = kScaled ? 1.0f : scales.at[2 * u + (r >> 4)];
#pragma unroll
                for (int k = 0; k < kSteps; k += 2) {
                    const u32x4 w = *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(
                        row + (((k + half) ^ R::key_place(r)) << 4));
                    const s16x8 a = T::from8(w[0], w[1], scale), b = T::from8(w[2], w[3], scale);
#pragma unroll
                    for (int t = 0; t < QT; ++t) {
                        s[t][u] = T::mfma(a, q[t][k], k == 0 ? f32x16{0} : s[t][u]);
                        s[t][u] = T::mfma(b, q[t][k + 1], s[t][u]);
                    }
                }
            } else {
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    const s16x8 a = *reinterpret_cast<const __attribute__((address_space(3))) s16x8*>(
                        row + (((2 * k + half) ^ R::key_place(r)) << 4));
#pragma unroll
                    for (int t = 0; t < QT; ++t) s[t][u] = T::mfma(a, q[t][k], k == 0 ? f32x16{0} : s[t][u]);
                }
            }
            if constexpr (kScaled) {
                const float low = scales.at[2 * u], high = scales.at[2 * u + 1];  // of keys 32 u + 0..15, 16..31
#pragma unroll
                for (int t = 0; t < QT; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[t][u][i] *= i < 8 ? low : high;
            }
        }
        s16x8 p[QT][NSUB][2], rest[QT][kScaled ? NSUB : 1][2];
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            if (kMasked) {
#pragma unroll
                for (int u = 0; u < NSUB; ++u) {
                    const uint32_t bits = allow[t][u] >> (4 * half);
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[t][u][i] = seen_or(bits, 8 * (i / 4) + i % 4, s[t][u][i]);
                }
            }
            // The maximum is not needed where the probabilities against the
            // one held stay in range: their sum, which is, tells. A row's own
            // sums (this lane's and that of the other half) decide for it
            // alone, so its bits do not depend on the wave's other rows.
            // (Against -inf, before a row's first visible key, they are infinite or NaN.)
            float sum = INFINITY;
            if (!__all(m[t] == -INFINITY)) sum = soften<NSUB>(s[t], p[t], rest[t], c, m[t] * c);
            const bool fits = sum <= kMostSum;
            if (__builtin_expect(!__all(fits), 0)) {
                raise<NSUB>(t, s[t], c, fits);
                sum = soften<NSUB>(s[t], p[t], rest[t], c, m[t] == -INFINITY ? 0.0f : m[t] * c);
            }
            l[t] += sum;
        }
        // Of 8 bits: row j of {0..3, 8..11} by two lanes, 8 bytes each.
        const int r = k8 ? (lane >> 1 & 3) + (lane & 8) : (lane & 15) >> 2;
        const lds_char* const first = values + (4 * half + r) * R::kBytes + (lane & 1) * 8;
        const int piece = k8 ? lane >> 4 & 1 : (lane >> 4 & 1) * 2 + (lane >> 1 & 1);
        uint32_t odd = 0;
#pragma unroll
        for (int u = 0; u < NSUB; ++u)
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int d = 0; d < kBlocks; ++d) {
                    s16x8 a = value(first, piece, r, u, k, d, scales);
                    if (kMasked) a = finite(a, odd);
#pragma unroll
                    for (int t = 0; t < QT; ++t) o[t][d] = P::mfma(a, p[t][u][k], o[t][d]);
                    if constexpr (kScaled) {
#pragma unroll
                        for (int t = 0; t < QT; ++t) o[t][d] = P::mfma(a, rest[t][u][k], o[t][d]);
                    }
                }
        if (kMasked && __any(odd != 0)) add_infinite<NSUB>(first, piece, r, half, allow, scales);
    }

    // A lane's probabilities 2^(c s - mc), packed for the second product (and
    // what that rounds off, where it is kept); returns their sum.
    template <int NSUB>
    static __device__ __forceinline__ float soften(const f32x16 (&s)[NSUB], s16x8 (&p)[NSUB][2], s16x8 (&rest)[kScaled ? NSUB : 1][2], float c,
                                                   float mc) {
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < NSUB; ++u)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                u32x4 w, v;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = exp2_fast(fmaf(s[u][8 * k + 2 * i], c, -mc)), y = exp2_fast(fmaf(s[u][8 * k + 2 * i + 1], c, -mc));
                    sum += x + y;
                    w[i] = P::pack(x, y);
                    if (kScaled) v[i] = P::pack(x - __uint_as_float(w[i] << 16), y - __uint_as_float(w[i] & 0xFFFF0000u));
                }
                p[u][k] = __builtin_bit_cast(s16x8, w);
                if (kScaled) rest[u][k] = __builtin_bit_cast(s16x8, v);
            }
        return sum;
    }

    // The maximum of tile t raised to that of its scores, the sums with it, for rows with a half that does not fit.
    template <int NSUB>
    __device__ __forceinline__ void raise(int t, const f32x16 (&s)[NSUB], float c, bool fits) {
        float top = s[0][0];
#pragma unroll
        for (int u = 0; u < NSUB; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][i]);
        top = max_halves(top);
        const bool rise = max_halves(fits ? 0.0f : 1.0f) > 0.0f && (top - m[t]) * c > kRise;  // false where both are -inf
        const float to = rise ? top : m[t];
        const float by = rise ? exp2_fast((m[t] - to) * c) : 1.0f;
        m[t] = to;
        l[t] *= by;
#pragma unroll
        for (int d = 0; d < kBlocks; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[t][d][i] *= by;
    }

    // V^T of keys 32 u + 16 k + {0..3, 8..11} (+ 4 in the upper half) and block d of columns.
    __device__ __forceinline__ s16x8 value(const lds_char* first, int piece, int r, int u, int k, int d, const TileScales& scales) {
        if constexpr (k8) {
            typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
            lds_char* const at = const_cast<lds_char*>(first) + (32 * u + 16 * k) * R::kBytes + (((2 * d + piece) ^ R::value_place(r)) << 4);
            const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)at);
            return Bf16::from8(w[0], w[1], scales.at[scales.blocks + 2 * u + k]);
        }
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        lds_char* const at = const_cast<lds_char*>(first) + (32 * u + 16 * k) * R::kBytes + (((4 * d + piece) ^ R::value_place(r)) << 4);
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 8 * R::kBytes));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }

    // A masked key has probability 0, but 0 * inf is not 0: infinities and
    // NaNs of V leave the product where keys are masked...
    static __device__ __forceinline__ s16x8 finite(s16x8 a, uint32_t& odd) {
        u32x4 w = __builtin_bit_cast(u32x4, a);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // Adding the exponent's lowest bit to it carries into the sign's place where all its bits are set.
            const uint32_t x = ((w[i] & P::kInf * 0x10001u) + (P::kInf & (0u - P::kInf)) * 0x10001u) & 0x80008000u;
            odd |= x;
            w[i] &= ~((x - (x >> 15)) | x);
        }
        return __builtin_bit_cast(s16x8, w);
    }

    // ...and come back for the queries that see them: a product of ones counts
    // the visible keys with +inf or NaN, and one those with -inf or NaN.
    // (Integer arithmetic on pairs throughout: as comparisons, this rare path
    // spilled scalar registers.)
    template <int NSUB>
    __device__ __forceinline__ void add_infinite(const lds_char* first, int piece, int r, int half, const uint32_t (&allow)[QT][NSUB],
                                                 const TileScales& scales) {
        constexpr uint32_t kPair = 0x10001u, kTop = 0x8000u * kPair;
#pragma nounroll
        for (int side = 0; side < 2; ++side) {
            const uint32_t sign = side ? kTop : 0u;
#pragma unroll
            for (int d = 0; d < kBlocks; ++d) {
                f32x16 n[QT];
#pragma unroll
                for (int t = 0; t < QT; ++t) n[t] = f32x16{0};
                int shift = 4 * half;
                asm volatile("" : "+v"(shift) : : "memory");  // nothing is worth keeping for the next block
#pragma unroll
                for (int u = 0; u < NSUB; ++u)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        u32x4 v = __builtin_bit_cast(u32x4, value(first, piece, r, u, k, d, scales));
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            // Top bits: at least inf; more (NaN); this sign. Then ones where they are set.
                            const uint32_t x = v[i] & ~kTop;
                            const uint32_t big = x + (0x8000u - P::kInf) * kPair, nan = x + (0x7FFFu - P::kInf) * kPair;
                            const uint32_t hit = big & (nan | ~(v[i] ^ sign)) & kTop;
                            v[i] = ((hit - (hit >> 15)) | hit) & P::kOne * kPair;
                        }
#pragma unroll
                        for (int t = 0; t < QT; ++t) {
                            const int bits = static_cast<int>(allow[t][u] >> (shift + 16 * k));
                            u32x4 w;
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int at = 8 * (i / 2) + 2 * (i % 2);
                                w[i] = (static_cast<uint32_t>(__builtin_amdgcn_sbfe(bits, at, 1)) & P::kOne) |
                                       (static_cast<uint32_t>(__builtin_amdgcn_sbfe(bits, at + 1, 1)) & P::kOne << 16);
                            }
                            n[t] = P::mfma(__builtin_bit_cast(s16x8, v), __builtin_bit_cast(s16x8, w), n[t]);
                        }
                    }
                const float add = side ? -INFINITY : INFINITY;
#pragma unroll
                for (int t = 0; t < QT; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[t][d][i] += n[t][i] > 0.0f ? add : 0.0f;
            }
        }
    }
};

// Bits 0..31 of the keys k0.. that a row sees which sees keys 0..end-1.
__device__ __forceinline__ uint32_t first_bits(int32_t n) {
    return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u;
}

// One lane's columns 8 * (i / 4) + 4 * half + i % 4 of block d, written as four elements at a time.
template <typename T>
__device__ __forceinline__ void store_four(uint16_t* to, float a, float b, float c, float d) {
    uint2 w;
    w.x = T::pack(a, b);
    w.y = T::pack(c, d);
    *reinterpret_cast<uint2*>(to) = w;
}

// --------------------------------------------------------------------------
// Packed prompts.
// --------------------------------------------------------------------------

struct PromptArgs {
    const uint16_t *q, *k, *v;
    uint16_t* out;
    float* lse;
    float* part_o;    // [place in the parts * heads + head][DP], where keys are split
    float2* part_ml;  // [the same]: c * maximum, sum
    const int32_t *q_offsets, *k_offsets;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;  // strides in elements
    int32_t n_seqs, heads, kv_heads, group, dim, n_q, n_k, n_slots;
    int32_t chunk, n_splits;  // keys of a part, parts of a sequence that holds every key
    int32_t part_rows;        // rows of all parts that the workspace holds
    bool all_fit;             // n_splits parts of every row
    float c, scale;
};

__device__ __forceinline__ int32_t bounded(int32_t x, int32_t most) { return x < 0 ? 0 : x > most ? most : x; }

// The last of n sequences whose place (of its number and first row) is at most
// `at`, by the whole wave: a search of single steps costs a memory latency for
// each, so it ends with the lanes looking at 64 sequences at once.
template <typename Place>
__device__ __forceinline__ int find_sequence(const int32_t* offsets, int n, int most, int at, int lane, Place place) {
    int lo = 0, hi = n - 1;
    while (hi - lo >= 64) {
        const int mid = (lo + hi + 1) / 2;
        if (place(mid, bounded(offsets[mid], most)) <= at) lo = mid; else hi = mid - 1;
    }
    const int b = lo + lane <= hi ? lo + lane : hi;
    const bool before = place(b, bounded(offsets[b], most)) <= at;
    // Places rise with b, so those at or before `at` are the first ones (lo is one of them, or nothing is).
    const int count = __popcll(__ballot(before && lo + lane <= hi));
    return __builtin_amdgcn_readfirstlane(lo + (count > 0 ? count - 1 : 0));
}

constexpr int kPromptKeys = 64;
constexpr int64_t kMostKeys = INT32_MAX - kPromptKeys;  // of a call: the first key after the last tile is an int32
constexpr int kPromptRows = 128;  // of a workgroup

// A sequence of a call, bounded to the buffers.
struct Prompt {
    int32_t q_begin, q_len, k_begin, k_len;
};

__device__ __forceinline__ Prompt prompt_of(const PromptArgs& A, int b) {
    Prompt p;
    p.q_begin = bounded(A.q_offsets[b], A.n_q), p.k_begin = bounded(A.k_offsets[b], A.n_k);
    const int32_t q_len = bounded(A.q_offsets[b + 1], A.n_q) - p.q_begin, k_len = bounded(A.k_offsets[b + 1], A.n_k) - p.k_begin;
    p.q_len = q_len > 0 ? q_len : 0, p.k_len = k_len > 0 ? k_len : 0;
    return p;
}

// Split prompts: sequence b's keys are cut into parts_in(k_len, chunk) parts,
// each a copy of the sequence's rows in the workspace, one sequence after the
// other. (A call that is split has at most 256 sequences and 2^15 rows, by
// plan_prompt, and a sequence at most 65 parts: sums of them fit 32 bits.)
__device__ __forceinline__ int32_t parts_in(int32_t k_len, int32_t chunk) { return k_len > chunk ? (k_len - 1) / chunk + 1 : 1; }

__device__ __forceinline__ int32_t part_rows_of(const Prompt& p, int32_t chunk) {
    const int32_t parts = parts_in(p.k_len, chunk);
    return parts > 1 ? p.q_len * parts : 0;
}

// Whether a sequence's parts, from its place on, lie in the workspace. They do
// unless offsets fall (sequences then lie over each other and need more rows than
// there are); such a sequence is left out.
__device__ __forceinline__ bool parts_fit(const PromptArgs& A, const Prompt& p, int32_t chunk, int32_t place) {
    return place + part_rows_of(p, chunk) <= A.part_rows;
}

template <int kLanes>
__device__ __forceinline__ int32_t sum_lanes(int32_t v) {
#pragma unroll
    for (int x = 1; x < kLanes; x *= 2) v += __shfl_xor(v, x);
    return v;
}

// Keys of a part: the host's number, which goes by the average sequence,
// doubled until every sequence's parts fit the workspace. kLanes neighbouring lanes call it together.
template <int kLanes>
__device__ __forceinline__ int32_t part_keys(const PromptArgs& A, int lane) {
    int32_t chunk = A.chunk;
    while (!A.all_fit) {
        int32_t rows = 0;
        for (int b = lane; b < A.n_seqs; b += kLanes) rows += part_rows_of(prompt_of(A, b), chunk);
        if (sum_lanes<kLanes>(rows) <= A.part_rows) break;
        chunk = chunk < 1 << 29 ? 2 * chunk : INT32_MAX;  // no sequence has more than INT32_MAX: the loop ends
    }
    return chunk;
}

// A workgroup of a split call: a tile of a sequence's rows and a part of its keys.
struct PromptPart {
    Prompt of;
    int32_t tile, tiles, part, parts;
    int32_t place;  // of the sequence's first row in the workspace
};

// The unit-th pair of a tile and a part, by a whole wave; false past the last.
__device__ __forceinline__ bool find_part(const PromptArgs& A, int32_t chunk, int32_t unit, int lane, PromptPart& to) {
    to.place = 0;
    for (int b0 = 0; b0 < A.n_seqs; b0 += 64) {
        const bool here = b0 + lane < A.n_seqs;
        const Prompt p = prompt_of(A, here ? b0 + lane : A.n_seqs - 1);
        const int32_t tiles = (p.q_len * A.group + kPromptRows - 1) / kPromptRows, parts = parts_in(p.k_len, chunk);
        const int32_t units = here ? tiles * parts : 0, rows = here ? part_rows_of(p, chunk) : 0;
        int32_t units_to = units, rows_to = rows;  // with the lanes before
        for (int x = 1; x < 64 && x < A.n_seqs; x *= 2) {
            const int32_t u = __shfl_up(units_to, x), r = __shfl_up(rows_to, x);
            if (lane >= x) units_to += u, rows_to += r;
        }
        const uint64_t past = __ballot(units_to > unit);
        if (past != 0) {
            const int at = __builtin_ctzll(past);
            auto of = [at](int32_t x) { return __builtin_amdgcn_readlane(x, at); };
            to.of = Prompt{of(p.q_begin), of(p.q_len), of(p.k_begin), of(p.k_len)};
            to.tiles = of(tiles), to.parts = of(parts);
            to.place += of(rows_to - rows);
            const int32_t i = unit - of(units_to - units);
            to.tile = i / to.parts, to.part = i % to.parts;
            return true;
        }
        unit -= __builtin_amdgcn_readlane(units_to, 63), to.place += __builtin_amdgcn_readlane(rows_to, 63);
    }
    return false;
}

// Bound by the SIMDs' instruction issue: with two waves a SIMD the matrix
// instructions hold 52% of its cycles and the softmax's ordinary ones 45%, LDS
// reads 26% (no bank conflicts). 16384 rows, 40 heads of 8, dim 128: 2.54-2.79
// ms by the card's clock, 986-1083 TFLOP/s of the products that are seen (a large
// matrix product reaches 1224). 64 rows a wave: 896; the next tile's scores
// computed beside this one's exponentials in one wave: 840; two groups of waves
// taking products and softmax in turn: 887-947; 8 waves sharing a tile: 984;
// tiles of 32 keys: 975 (when this form reached 1015-1045).
// Workgroup: one sequence and key/value head, 32 * QT * NW rows of its group
// of heads: row r is head r % group of position r / group. Rows of one position
// see the same keys, so a workgroup's rows reach over few positions: the tiles
// on the causal edge waste less, and short prompts fill their last workgroup
// (12 prompts of 85-1999 rows, 5 heads a group: 10% fewer tiles than with rows
// of one head).
// Slots: sequence b's tiles of rows start at slot first_row / rows + b, a place
// that needs no sums over the sequences before it; slots past a sequence's
// rows are empty. Later slots, whose rows see more keys, start first.
// Parts: where a call has few rows and many keys (the next piece of a prompt
// over a long context) each workgroup takes a part of its rows' keys, and
// prompt_join_kernel joins them. The sums lie one sequence after the other, so
// that a short sequence has none for a long one's parts, and only pairs of a
// tile and a part that exist are workgroups (32 prompts of 112 rows over 2112
// keys, 8 heads of 1: 62 us and 67 MB; with the longest possible sequence's
// parts for each row 93 us and 939 MB. Four small ones: 15.2 us, 14.5.)
template <typename T, int DP, int QT, int NW, bool kParts>
__global__ __launch_bounds__(64 * NW, QT == 1 && DP <= 128 ? 2 : 1) void prompt_kernel(const PromptArgs A) {
    typedef Rows<DP> R;
    constexpr int KT = DP <= 128 ? kPromptKeys : 32;
    constexpr int NSUB = KT / 32;
    constexpr int BM = 32 * QT * NW;
    constexpr int kTile = KT * R::kBytes;            // bytes of a tile of K, and of V
    constexpr int kLoads = kTile / 1024 / NW;        // loads a wave makes of either
    __shared__ __attribute__((aligned(1024))) char lds[4 * kTile];
    lds_char* const shared = (lds_char*)lds;

    // Consecutive workgroups take the key/value heads in turn: with eight of
    // them an XCD keeps to one head, whose keys and values stay in its L2.
    const int kvh = blockIdx.x % A.kv_heads;
    const int group = A.group;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int q_begin, q_len, k_begin, k_len, rows, row0;
    int split = 0, chunk = 0, place = 0;
    if constexpr (kParts) {
        chunk = __builtin_amdgcn_readfirstlane(part_keys<64>(A, lane));
        PromptPart p;
        if (!find_part(A, chunk, static_cast<int32_t>(blockIdx.x / A.kv_heads), lane, p)) return;
        place = __builtin_amdgcn_readfirstlane(p.place);
        if (!parts_fit(A, p.of, chunk, place)) return;
        q_begin = p.of.q_begin, q_len = p.of.q_len, k_begin = p.of.k_begin, k_len = p.of.k_len;
        rows = q_len * group, row0 = (p.tiles - 1 - p.tile) * BM;
        split = p.part;
    } else {
        const int slot = A.n_slots - 1 - static_cast<int>(blockIdx.x / A.kv_heads);
        const int lo = find_sequence(A.q_offsets, A.n_seqs, A.n_q, slot, lane, [&](int b, int first) { return first * group / BM + b; });
        const int q_end = bounded(A.q_offsets[lo + 1], A.n_q), k_end = bounded(A.k_offsets[lo + 1], A.n_k);
        q_begin = bounded(A.q_offsets[lo], A.n_q), k_begin = bounded(A.k_offsets[lo], A.n_k);
        q_len = q_end - q_begin, k_len = k_end > k_begin ? k_end - k_begin : 0;
        rows = q_len * group;
        row0 = (slot - (q_begin * group / BM + lo)) * BM;
        if (row0 < 0 || row0 >= rows) return;
    }

    const int half = lane >> 5;
    const int shift = k_len - q_len;  // position i sees keys 0 .. i + shift
    const int wave_row = row0 + wave * 32 * QT;
    auto seen_by = [&](int row) { return row / group + 1 + shift < 0 ? 0 : row / group + 1 + shift; };

    const int keys_wg = seen_by((row0 + BM < rows ? row0 + BM : rows) - 1);  // keys that some row here sees
    const int begin = kParts ? split * chunk : 0;  // at most k_len
    if (split > 0 && begin >= keys_wg) return;
    const bool parted = kParts && keys_wg > chunk;
    const int end = !kParts || keys_wg - begin < chunk ? keys_wg : begin + chunk;
    int keys_wave = wave_row >= rows ? 0 : seen_by((wave_row + 32 * QT < rows ? wave_row + 32 * QT : rows) - 1);
    keys_wave = keys_wave < end ? keys_wave : end;

    const uint16_t* const k_base = A.k + k_begin * A.k_row + kvh * A.k_head;
    const uint16_t* const v_base = A.v + k_begin * A.v_row + kvh * A.v_head;
    const int pieces = A.dim / 8 - 1;  // the last 16-byte piece of a row; pieces past it repeat it at first
    const int lane_row = lane / R::kPieces, lane_piece = lane % R::kPieces;
    const uint32_t k_bytes = static_cast<uint32_t>(2 * A.k_row), v_bytes = static_cast<uint32_t>(2 * A.v_row);
    auto load_tile = [&](int k0, lds_char* to) {
        // Rows past the last key repeat it; no row sees them.
        const int last = k_len - 1 - k0;
        const bool whole = last >= KT - 1;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int load = wave * kLoads + i;
            const int r0 = load * R::kPerLoad, r = r0 + lane_row;
            const int kx = lane_piece ^ R::key_place(r), vx = lane_piece ^ R::value_place(r);
            const uint32_t kp = (kx < pieces ? kx : pieces) * 16, vp = (vx < pieces ? vx : pieces) * 16;
            const int from0 = whole ? r0 : 0;
            const uint32_t from = whole ? lane_row : (r < last ? r : last);
            const char* const kb = reinterpret_cast<const char*>(k_base + (k0 + from0) * A.k_row);
            const char* const vb = reinterpret_cast<const char*>(v_base + (k0 + from0) * A.v_row);
            load_to_lds(kb + (from * k_bytes + kp), to + load * 1024);
            load_to_lds(vb + (from * v_bytes + vp), to + kTile + load * 1024);
        }
    };
    if (begin < end) load_tile(begin, shared);
    State<T, DP, QT> st;
    st.clear();
    int32_t sees[QT];  // keys that the lane's rows see
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int row = wave_row + 32 * t + (lane & 31);
        const int at = row < rows ? row : rows - 1;
        st.load_query(t, A.q + (q_begin + at / group) * A.q_row + (kvh * group + at % group) * A.q_head, A.dim, half);
        sees[t] = seen_by(at);
    }
    auto arrived = [&](lds_char* to) __attribute__((always_inline)) {
        wait_loads<0>();
        if (A.dim < DP) clear_past<R, KT / NW>(A.dim / 8, to, wave * (KT / NW), lane);
        __syncthreads();
    };
    arrived(shared);
    int k0 = begin;
    uint32_t at = 0;  // the tile's place in LDS
    // Tiles that every row of the workgroup sees whole, then those it needs
    // masks for. The two places are passed as restrict pointers: the compiler
    // then knows that reads of a tile need not wait for the loads of the next.
    for (const int whole = row0 / group + 1 + shift; k0 + KT <= whole && k0 < end; k0 += KT, at ^= 2 * kTile) {
        auto tile = [&](lds_char* __restrict__ next, const lds_char* __restrict__ now) __attribute__((always_inline)) {
            if (k0 + KT < end) load_tile(k0 + KT, next);
            const uint32_t all[QT][NSUB] = {};
            st.template step<NSUB, false>(now, now + kTile, A.c, lane, all);
        };
        tile(shared + (at ^ 2 * kTile), shared + at);
        arrived(shared + (at ^ 2 * kTile));
    }
    for (; k0 < end; k0 += KT, at ^= 2 * kTile) {
        auto tile = [&](lds_char* __restrict__ next, const lds_char* __restrict__ now) __attribute__((always_inline)) {
            if (k0 + KT < end) load_tile(k0 + KT, next);
            if (k0 < keys_wave) {
                uint32_t allow[QT][NSUB];
#pragma unroll
                for (int t = 0; t < QT; ++t)
#pragma unroll
                    for (int u = 0; u < NSUB; ++u) allow[t][u] = first_bits(sees[t] - k0 - 32 * u);
                st.template step<NSUB, true>(now, now + kTile, A.c, lane, allow);
            }
        };
        tile(shared + (at ^ 2 * kTile), shared + at);
        arrived(shared + (at ^ 2 * kTile));
    }

#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int r = wave_row + 32 * t + (lane & 31);
        const float l = add_halves(st.l[t]);
        if (r >= rows) continue;
        const int row = q_begin + r / group, head = kvh * group + r % group;
        const int64_t rh = static_cast<int64_t>(row) * A.heads + head;
        const int64_t part = (place + split * q_len + r / group) * static_cast<int64_t>(A.heads) + head;
        const float by = parted ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
        uint16_t* const to = A.out + row * A.out_row + head * A.out_head;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int x = 32 * d + 8 * i + 4 * half;
                const f32x16& o = st.o[t][d];
                if (parted)
                    *reinterpret_cast<float4*>(A.part_o + part * DP + x) = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                else if (x < A.dim)
                    store_four<T>(to + x, o[4 * i] * by, o[4 * i + 1] * by, o[4 * i + 2] * by, o[4 * i + 3] * by);
            }
        if (half != 0) continue;
        if (parted) A.part_ml[part] = make_float2(st.m[t] * A.c, l);
        else if (A.lse != nullptr) A.lse[rh] = l == 0.0f ? -INFINITY : st.m[t] * A.scale + logf(l);
    }
}

// One row and head's parts in their order, by DP / 4 threads with four columns
// each: part s at s * all + rh.
template <typename T, int DP>
__device__ __forceinline__ void join_parts(const float* part_o, const float2* part_ml, int64_t all, int64_t rh, int parts, int col,
                                           int dim, uint16_t* to, float* lse) {
    constexpr int kCols = DP / 4;
    float top = -INFINITY;
    for (int s = col; s < parts; s += kCols) top = fmaxf(top, part_ml[s * all + rh].x);
#pragma unroll
    for (int x = 1; x < kCols; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
    float l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s0 = 0; s0 < parts; s0 += 4) {
        float2 ml[4];
        float4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int s = s0 + i < parts ? s0 + i : s0;
            ml[i] = part_ml[s * all + rh];
            v[i] = *reinterpret_cast<const float4*>(part_o + (s * all + rh) * DP + 4 * col);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (s0 + i >= parts || ml[i].y == 0.0f) continue;  // a part without a visible key (NaN scores leave a NaN sum)
            const float by = exp2_fast(ml[i].x - top);
            l += ml[i].y * by;
            o.x += v[i].x * by, o.y += v[i].y * by, o.z += v[i].z * by, o.w += v[i].w * by;
        }
    }
    const float by = l == 0.0f ? 0.0f : 1.0f / l;
    if (4 * col < dim) store_four<T>(to + 4 * col, o.x * by, o.y * by, o.z * by, o.w * by);
    if (col == 0 && lse != nullptr) *lse = l == 0.0f ? -INFINITY : top * (1.0f / kLog2E) + logf(l);
}

// The parts of split prompts; a row's number of parts follows from its workgroup's keys.
template <typename T, int DP>
__global__ __launch_bounds__(256) void prompt_join_kernel(const PromptArgs A) {
    constexpr int kCols = DP / 4, kSides = 256 / kCols;
    const int64_t all = static_cast<int64_t>(A.n_q) * A.heads;
    const int64_t rh = static_cast<int64_t>(blockIdx.x) * kSides + threadIdx.x / kCols;
    if (rh >= all) return;
    const int row = static_cast<int>(rh / A.heads), head = static_cast<int>(rh % A.heads);
    int lo = 0;
    for (int hi = A.n_seqs - 1; lo < hi;) {
        const int mid = (lo + hi + 1) / 2;
        if (bounded(A.q_offsets[mid], A.n_q) <= row) lo = mid; else hi = mid - 1;
    }
    const Prompt p = prompt_of(A, lo);
    if (row < p.q_begin || row >= p.q_begin + p.q_len) return;
    const int col = threadIdx.x % kCols;
    const int32_t chunk = part_keys<kCols>(A, col);
    // The keys of the row's workgroup decide its parts.
    const int rows = p.q_len * A.group, r = (row - p.q_begin) * A.group + head % A.group;
    const int row0 = r / kPromptRows * kPromptRows;
    const int last = (row0 + kPromptRows < rows ? row0 + kPromptRows : rows) - 1;
    const int keys = last / A.group + 1 + p.k_len - p.q_len;
    if (keys <= chunk) return;
    int32_t place = 0;
    if (lo > 0) {
        for (int b = col; b < lo; b += kCols) place += part_rows_of(prompt_of(A, b), chunk);
        place = sum_lanes<kCols>(place);
    }
    if (!parts_fit(A, p, chunk, place)) return;
    place += row - p.q_begin;
    join_parts<T, DP>(A.part_o, A.part_ml, static_cast<int64_t>(p.q_len) * A.heads, static_cast<int64_t>(place) * A.heads + head,
                      (keys - 1) / chunk + 1, col, A.dim, A.out + row * A.out_row + head * A.out_head,
                      A.lse != nullptr ? A.lse + rh : nullptr);
}

constexpr int64_t kPromptScratch = 64 << 20;  // bytes of split prompts' sums that need no further reason

int padded_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// Keys of a part. 512 workgroups run at a time; a call with up to half as many
// splits its keys to fill them, where the keys are enough to pay for writing
// and joining the parts' sums: 8 a workgroup of the call, and 512. (40 heads of
// 8, dim 128, us with and without the split: 50 rows over 800 keys 17, 25; 50
// over 12000 33, 257; 400 over 1500 33, 40; 400 over 800 29, 25 and so not
// split; 800 over 3000 66, 71; 800 over 1500 45, 40 and so not split; 1100 over
// 3000 101, 77. Twice as many parts: 400 over 3000 51, not 43.)
void plan_prompt(PromptArgs& A, int64_t n_rows, int64_t n_keys) {
    const int64_t groups = (n_rows * A.group / kPromptRows + A.n_seqs) * A.kv_heads;
    const int64_t each = A.n_seqs > 0 ? n_keys / A.n_seqs : 0;  // keys of a sequence, about
    int64_t chunk = INT32_MAX;  // no call has more keys
    if (groups <= 256 && each > 512 && each > 8 * groups) {
        const int64_t parts = 512 / (groups > 0 ? groups : 1);
        chunk = each / parts > 256 ? each / parts : 256;
        if (n_keys / chunk >= 64) chunk = n_keys / 64 + 1;  // sequences far longer than the others
        chunk = (chunk + 63) / 64 * 64;
    }
    A.chunk = static_cast<int32_t>(chunk);
    A.n_splits = n_keys > chunk ? static_cast<int32_t>((n_keys + chunk - 1) / chunk) : 1;
    // Rows of parts: what one sequence needs with every key; of several, which
    // are shorter, twice what they need if all are of one length, or 64 MiB.
    // (The kernels take longer parts where that is too little: lengths are on
    // the GPU. With as many rows as n_splits parts of every row, 32 prompts of
    // 112 rows over 2112 keys took 939 MB for the 30 they use.)
    const int64_t row = static_cast<int64_t>(A.kv_heads) * A.group * (4 * padded_dim(A.dim) + 8);
    const int64_t even = 2 * n_rows * ((each + chunk - 1) / chunk), least = kPromptScratch / row;
    const int64_t most = n_rows * A.n_splits, rows = even > least ? even : least;
    A.part_rows = A.n_splits > 1 ? static_cast<int32_t>(most < rows ? most : rows) : 0;
    A.all_fit = most <= rows;
}

template <typename T, int DP>
int launch_prompt(PromptArgs& A, hipStream_t s) {
    constexpr int QT = 1, NW = 4, BM = 32 * QT * NW;
    static_assert(BM == kPromptRows, "the join goes by the same rows");
    const int64_t rows = static_cast<int64_t>(A.n_q) * A.group;
    // Split: a sequence's tiles are its rows / BM and one at most, in each of its
    // parts; the parts are one for each chunk and sequence at most, their rows
    // at most part_rows. Sequences of one part have the other tiles.
    int64_t units = rows / BM + A.n_seqs;
    if (A.n_splits > 1)
        units = A.n_seqs == 1 ? (rows + BM - 1) / BM * A.n_splits
                              : units + static_cast<int64_t>(A.part_rows) * A.group / BM + A.n_k / A.chunk + A.n_seqs;
    const int64_t groups = units * A.kv_heads;
    if (rows > INT32_MAX || groups > INT32_MAX) return fail(AIMG_ERR_UNSUPPORTED, "prompt attention: too many rows times heads");
    A.n_slots = static_cast<int32_t>(rows / BM + A.n_seqs);
    const dim3 grid(static_cast<uint32_t>(groups)), block(64 * NW);
    if (A.n_splits == 1) {
        hipLaunchKernelGGL((prompt_kernel<T, DP, QT, NW, false>), grid, block, 0, s, A);
    } else {
        hipLaunchKernelGGL((prompt_kernel<T, DP, QT, NW, true>), grid, block, 0, s, A);
        constexpr int kRows = 1024 / DP;
        const int64_t all = static_cast<int64_t>(A.n_q) * A.heads;
        hipLaunchKernelGGL((prompt_join_kernel<T, DP>), dim3(static_cast<uint32_t>((all + kRows - 1) / kRows)), dim3(256), 0, s, A);
    }
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess)
        return fail(AIMG_ERR_HIP, std::string("kernel launch failed: ") + hipGetErrorString(err));
    return AIMG_OK;
}

// --------------------------------------------------------------------------
// Drafted tokens over a paged cache.
// --------------------------------------------------------------------------

struct TreeArgs {
    const uint16_t* q;
    const char *k, *v;
    const float *k_scales, *v_scales;                // of a cache in 8 bits: [page][head][block], the last contiguous
    int64_t scale_page, scale_head;                  // strides
    uint16_t* out;
    float* lse;
    const int32_t *table, *lengths, *seqs, *offsets;
    const uint64_t* masks;
    float* part_o;    // [split][row * heads + head][DP]
    float2* part_ml;  // [split][row * heads + head]: c * maximum, sum
    int64_t q_row, q_head, out_row, out_head, page_stride, slot_stride, kv_head_stride;  // in elements
    int32_t table_stride, max_pages, n_slots, n_pages, page_size, n_seqs, heads, kv_heads, dim, n_q, words;
    int32_t max_drafts, chunk, n_splits, row_blocks;
    uint32_t magic;   // 2^32 / page_size, for divisions by it
    float c, scale;
};

// key / page_size and key % page_size. The product is off by less than one
// either way (key below 2^31, magic at most 1 below or above 2^32 / page_size).
__device__ __forceinline__ void page_of(const TreeArgs& A, int32_t key, int32_t& page, int32_t& slot) {
    int32_t p = static_cast<int32_t>(__umulhi(static_cast<uint32_t>(key), A.magic));
    int32_t r = key - p * A.page_size;
    if (r < 0) --p, r += A.page_size;
    if (r >= A.page_size) ++p, r -= A.page_size;
    page = p, slot = r;
}

// A sequence of the call: its drafted rows and the positions it holds. What
// the arrays say is bounded to the buffers.
struct Drafted {
    int32_t row, n, context, end;  // first row of q, drafted tokens, positions before and with them
    const int32_t* pages;
};

__device__ __forceinline__ Drafted drafted(const TreeArgs& A, int b) {
    Drafted d;
    d.row = bounded(A.offsets[b], A.n_q);
    const int32_t last = bounded(A.offsets[b + 1], A.n_q);
    d.n = bounded(last - d.row, A.max_drafts);
    const int32_t slot = A.seqs[b];
    const bool known = slot >= 0 && slot < A.n_slots;
    const int64_t most = static_cast<int64_t>(A.max_pages) * A.page_size;
    if (d.n > most) d.n = static_cast<int32_t>(most);
    d.context = known ? bounded(A.lengths[slot], static_cast<int32_t>(most - d.n)) : 0;
    d.end = known ? d.context + d.n : 0;
    d.pages = A.table + static_cast<int64_t>(known ? slot : 0) * A.table_stride;
    return d;
}

// Bits of the keys k0 .. k0 + 31 that drafted token t (row of q: row) sees.
__device__ __forceinline__ uint32_t seen_keys(const TreeArgs& A, const Drafted& D, int row, int t, int k0) {
    const int32_t j = k0 - D.context;  // drafted index of the first key, negative: so many keys of context
    if (j <= -32) return ~0u;
    const int32_t at = j < 0 ? 0 : j;
    uint32_t bits;
    if (A.masks == nullptr) {
        bits = first_bits(t + 1 - at);
    } else {
        const int32_t w = at >> 6, sh = at & 63;
        const uint64_t* const m = A.masks + static_cast<int64_t>(row) * A.words;
        uint64_t v = w < A.words ? m[w] >> sh : 0;
        if (sh > 32 && w + 1 < A.words) v |= m[w + 1] << (64 - sh);
        bits = static_cast<uint32_t>(v) & first_bits(D.n - at);
    }
    return j < 0 ? bits << -j | first_bits(-j) : bits;
}

// One call's rows of a (sequence, key/value head): drafted token t and head g
// of the group are row t * group + g, so a key and value are read once for all
// of them. kShared: NW waves with 32 * QT rows each share tiles of K and V.
// Otherwise the waves hold the same 32 * QT rows and take tiles in turn, each
// into its own part of LDS with no barrier in the loop, and join their sums at
// the end: one token's group (5 rows of 32 here) leaves the matrix cores idle,
// but the bytes in flight, not the products, bound it.
// Bound by HBM where contexts are long: 16 trees of 4-16 tokens over 9000-65000
// positions, 40 heads of 8, dim 128, read 1.73 GB in 330 us, 5.2 TB/s; 64
// single tokens over 2000-8000 5.1 TB/s. 8 trees of 1-33 tokens over 700-6000
// positions take 27 us, 3.7 TB/s: 368 workgroups have rows and keys, fewer than
// the 512 that run at a time, and each has ten tiles at most between its first
// loads and its sums. Without masks, too, every block of rows takes all keys of
// its sequence: right, but for a long stretch of a prompt over the cache twice
// the products it needs (4096 rows over no context 521 us, packed prompts 204;
// over 8000 positions 1285 and 852).
// kPages: what of a tile never crosses a page, and so has one base address: 2
// the tile, 1 the rows of one load (2 to 8), 0 a row. (With addresses made lane
// by lane for pages of 16, 54 trees over 139-2238 positions took 155 us.)
// k8: a cache in 8 bits, whose codes become elements in every wave that reads
// them. Each wave brings its tile's scales along, a load of 4 bytes a lane into
// a place of its own. 64 single tokens over 1900-8100 positions 113 us, 4.8 TB/s.
// Shared tiles, 16 trees of 4-16 tokens over 9000-65000 313 us, 3.8 TB/s: matrix
// units 19% and vector instructions 28% of the cycles, for the workgroups' rows
// follow from the largest tree (128, 80 of them used) and of the waves, by their
// keys, 48% hold rows of their sequence; the others load and wait. (Elements
// formed once for all waves, in LDS, between two barriers: 391 us, not 330 with
// the same parts; a lane's places in its loads worked out for every tile: 352.)
// Of dim 64, 96 and 256 (16 heads of 4), 64 single tokens 4.9, 3.8 and 2.6 TB/s,
// over 16 bits 4.7, 4.5 and 4.3.
template <typename T, int DP, int QT, int NW, bool kShared, int kPages, bool k8>
__global__ __launch_bounds__(64 * NW, QT == 1 && DP <= 128 ? 2 : 1) void tree_kernel(const TreeArgs A) {
    typedef State<T, DP, QT, k8> St;
    typedef typename St::R R;
    constexpr int kSize = k8 ? 1 : 2;  // bytes of an element
    constexpr int KT = kShared && DP <= 128 ? 64 : 32;
    constexpr int NSUB = KT / 32;
    constexpr int kTile = KT * R::kBytes;
    constexpr int kLoads = kTile / 1024 / (kShared ? NW : 1);  // loads a wave makes of K, and of V
    constexpr int kBlocks = KT / kBlock;                       // of a tile
    constexpr int kScales = k8 ? 2 * NW * 256 : 0;             // bytes of two tiles' scales for each wave
    constexpr int BM = 32 * QT * (kShared ? NW : 1);
    constexpr int kRow = DP + 4;  // floats of a row of sums in LDS: 16 bytes more than a multiple of all banks
    constexpr int kSums = kShared ? 0 : NW * 32 * QT * (kRow * 4 + 8);
    constexpr int kTiles = 4 * kTile * (kShared ? 1 : NW);
    __shared__ __attribute__((aligned(1024))) char lds[kTiles + kScales > kSums ? kTiles + kScales : kSums];

    const int group = A.heads / A.kv_heads;
    int id = blockIdx.x;
    const int kvh = id % A.kv_heads;
    id /= A.kv_heads;
    const int split = id % A.n_splits;
    id /= A.n_splits;
    const int block = id % A.row_blocks, b = id / A.row_blocks;
    const Drafted D = drafted(A, b);
    const int rows = D.n * group;
    if (block * BM >= rows) return;
    const int lo = split * A.chunk;
    // The last part takes what a sequence holds beyond the longest one planned for.
    const int hi = split == A.n_splits - 1 || D.end - lo < A.chunk ? D.end : lo + A.chunk;
    if (split > 0 && lo >= hi) return;  // the join knows how many parts a sequence has

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int half = lane >> 5;
    lds_char* const mine = (lds_char*)lds + (kShared ? 0 : wave * 4 * kTile);

    const int pieces = A.dim * kSize / 16 - 1;
    const int lane_row = lane / R::kPieces, lane_piece = lane % R::kPieces;
    const uint32_t row_bytes = static_cast<uint32_t>(kSize * A.slot_stride);
    const int64_t head_at = kvh * A.kv_head_stride;
    lds_char* const scales = (lds_char*)lds + kTiles + wave * 512;
    const int lane_block = lane % kBlocks;
    const float* const lane_scales = !k8 ? nullptr : (lane / kBlocks % 2 == 0 ? A.k_scales : A.v_scales) + kvh * A.scale_head;
    const int load0 = kShared ? wave * kLoads : 0;
    // A lane holds the number of page `first_page` + lane of the sequence, for
    // 64 pages at a time: a tile's page numbers then come out of a register,
    // and no load of the loop waits for another.
    int32_t first_page = 0, held = 0;
    auto hold = [&](int32_t page) __attribute__((always_inline)) {
        first_page = page;
        const int32_t at = page + lane < A.max_pages ? page + lane : A.max_pages - 1;
        const int32_t id = D.pages[at];
        held = static_cast<uint32_t>(id) < static_cast<uint32_t>(A.n_pages) ? id : 0;
    };
    // The scales of the blocks of keys k0 .., those past the last key's being its own.
    auto load_scales = [&](int k0, int last, lds_char* to) __attribute__((always_inline)) {
        const int at = kBlock * lane_block;
        int32_t p, slot;
        page_of(A, k0 + (at < last ? at : last), p, slot);
        const int64_t id = __builtin_amdgcn_ds_bpermute(4 * (p - first_page), held);
        load4_to_lds(lane_scales + (id * A.scale_page + slot / kBlock), to);
    };
    // A lane's place in each of its loads.
    uint32_t k_off[k8 ? kLoads : 1], v_off[k8 ? kLoads : 1];
    const char* const k_head = A.k + kSize * head_at;
    const char* const v_head = A.v + kSize * head_at;
    if constexpr (k8) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int r = (load0 + i) * R::kPerLoad + lane_row;
            const int kx = lane_piece ^ R::key_place(r), vx = lane_piece ^ R::value_place(r);
            k_off[i] = lane_row * row_bytes + (kx < pieces ? kx : pieces) * 16;
            v_off[i] = lane_row * row_bytes + (vx < pieces ? vx : pieces) * 16;
        }
    }
    // Keys past the last one repeat it; no row sees them.
    auto issue = [&](int k0, lds_char* to, lds_char* to_scales) __attribute__((always_inline)) {
        const int last = D.end - 1 - k0 < KT - 1 ? D.end - 1 - k0 : KT - 1;
        int32_t page, first, page_end, unused;
        page_of(A, k0, page, first);
        page_of(A, k0 + last, page_end, unused);
        if (page_end >= first_page + 64) hold(page);
        if (k8 && kPages > 0 && last == KT - 1) {
            // A whole tile: uniform addresses, and offsets that a lane keeps.
            const int32_t id = __builtin_amdgcn_readlane(held, page - first_page);
            if (kPages == 2) load4_to_lds(lane_scales + (id * A.scale_page + static_cast<uint32_t>(first) / kBlock) + lane_block, to_scales);
            else load_scales(k0, last, to_scales);
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                int64_t from = id * A.page_stride + (first + (load0 + i) * R::kPerLoad) * A.slot_stride;
                if (kPages == 1) {
                    int32_t p, slot;
                    page_of(A, k0 + (load0 + i) * R::kPerLoad, p, slot);
                    from = __builtin_amdgcn_readlane(held, p - first_page) * A.page_stride + slot * A.slot_stride;
                }
                load_to_lds(k_head + from + k_off[i], to + (load0 + i) * 1024);
                load_to_lds(v_head + from + v_off[i], to + kTile + (load0 + i) * 1024);
            }
            return;
        }
        int64_t tile_at = 0;
        if (kPages == 2)
            tile_at = kSize * (__builtin_amdgcn_readlane(held, page - first_page) * A.page_stride + first * A.slot_stride + head_at);
        if constexpr (k8) load_scales(k0, last, to_scales);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int load = load0 + i;
            const int r0 = load * R::kPerLoad, r = r0 + lane_row;
            const int kx = lane_piece ^ R::key_place(r), vx = lane_piece ^ R::value_place(r);
            const uint32_t kp = (kx < pieces ? kx : pieces) * 16, vp = (vx < pieces ? vx : pieces) * 16;
            int64_t at = tile_at;
            uint32_t from = r < last ? r : last;
            if (kPages == 1) {
                const int row = r0 < last ? r0 : last;
                int32_t p, slot;
                page_of(A, k0 + row, p, slot);
                at = kSize * (__builtin_amdgcn_readlane(held, p - first_page) * A.page_stride + slot * A.slot_stride + head_at);
                from -= row;
            } else if (kPages == 0) {
                int32_t p, slot;
                page_of(A, k0 + from, p, slot);
                const int64_t id = __builtin_amdgcn_ds_bpermute(4 * (p - first_page), held);
                at = kSize * (id * A.page_stride + slot * A.slot_stride + head_at);
                from = 0;
            }
            load_to_lds(A.k + at + (from * row_bytes + kp), to + load * 1024);
            load_to_lds(A.v + at + (from * row_bytes + vp), to + kTile + load * 1024);
        }
    };

    // A wave whose rows are past the last only loads.
    const bool active = !kShared || block * BM + wave * 32 * QT < rows;
    constexpr int kStep = kShared ? KT : KT * NW;
    int k0 = lo + (kShared ? 0 : wave * KT);
    uint32_t at = 0;
    if (k0 < hi) {
        int32_t page, unused;
        page_of(A, k0, page, unused);
        hold(page);
        issue(k0, mine, scales);
    }
    St st;
    st.clear();
    int token[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        int r = block * BM + (kShared ? wave * 32 * QT : 0) + 32 * t + (lane & 31);
        r = r < rows ? r : rows - 1;
        token[t] = r / group;
        st.load_query(t, A.q + (D.row + token[t]) * A.q_row + (kvh * group + r % group) * A.q_head, A.dim, half);
    }
    auto arrived = [&](lds_char* to) __attribute__((always_inline)) {
        wait_loads<0>();
        if (A.dim < DP) clear_past<R, KT / NW>(A.dim * kSize / 16, to, wave * (KT / NW), lane);
        __syncthreads();
    };
    if (kShared) arrived(mine);
    // Two tiles in turn.
    auto tile = [&](auto masked, lds_char* __restrict__ next, lds_char* __restrict__ now, lds_char* __restrict__ next_scales,
                    lds_char* __restrict__ now_scales) __attribute__((always_inline)) {
        constexpr bool kMasked = decltype(masked)::value;
        const bool more = k0 + kStep < hi;
        if (more) issue(k0 + kStep, next, next_scales);
        if (!kShared) {
            // All but the loads just issued, the next tile's, have arrived. The
            // tile's reads take their place from the wait, so that none can
            // move before it.
            uint32_t zero = 0;
            if (more) asm volatile("s_waitcnt vmcnt(%1)" : "+v"(zero) : "n"(2 * kLoads + (k8 ? 1 : 0)) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" : "+v"(zero) : : "memory");
            now += zero;
            now_scales += zero;
            if (A.dim < DP) clear_past<R, KT>(A.dim * kSize / 16, now, 0, lane);
        }
        if (!active) return;
        uint32_t allow[QT][NSUB] = {};
        if (kMasked) {
#pragma unroll
            for (int t = 0; t < QT; ++t)
#pragma unroll
                for (int u = 0; u < NSUB; ++u) allow[t][u] = seen_keys(A, D, D.row + token[t], token[t], k0 + 32 * u);
        }
        typename St::TileScales tile_scales;
        if constexpr (k8) tile_scales = {reinterpret_cast<const __attribute__((address_space(3))) float*>(now_scales), kBlocks};
        st.template step<NSUB, kMasked>(now, now + kTile, A.c, lane, allow, tile_scales);
    };
    uint32_t at_scales = 0;
    for (; k0 + KT <= D.context && k0 < hi; k0 += kStep, at ^= 2 * kTile, at_scales ^= 256) {
        tile(std::integral_constant<bool, false>{}, mine + (at ^ 2 * kTile), mine + at, scales + (at_scales ^ 256), scales + at_scales);
        if (kShared) arrived(mine + (at ^ 2 * kTile));
    }
    for (; k0 < hi; k0 += kStep, at ^= 2 * kTile, at_scales ^= 256) {
        tile(std::integral_constant<bool, true>{}, mine + (at ^ 2 * kTile), mine + at, scales + (at_scales ^ 256), scales + at_scales);
        if (kShared) arrived(mine + (at ^ 2 * kTile));
    }

    const int64_t part = static_cast<int64_t>(split) * A.n_q * A.heads;
    const bool parted = A.n_splits > 1 && D.end > A.chunk;  // the join leaves sequences of one part alone
    if (kShared) {
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            const int r = block * BM + wave * 32 * QT + 32 * t + (lane & 31);
            const float l = add_halves(st.l[t]);
            if (r >= rows) continue;
            const int row = D.row + token[t], head = kvh * group + r % group;
            const int64_t rh = static_cast<int64_t>(row) * A.heads + head;
            const float by = parted ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
            uint16_t* const to = A.out + row * A.out_row + head * A.out_head;
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int x = 32 * d + 8 * i + 4 * half;
                    const f32x16& o = st.o[t][d];
                    if (parted)
                        *reinterpret_cast<float4*>(A.part_o + (part + rh) * DP + x) = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    else if (x < A.dim)
                        store_four<T>(to + x, o[4 * i] * by, o[4 * i + 1] * by, o[4 * i + 2] * by, o[4 * i + 3] * by);
                }
            if (half == 0) {
                if (parted) A.part_ml[part + rh] = make_float2(st.m[t] * A.c, l);
                else if (A.lse != nullptr) A.lse[rh] = l == 0.0f ? -INFINITY : st.m[t] * A.scale + logf(l);
            }
        }
        return;
    }

    // The waves' sums, joined in LDS.
    __syncthreads();
    float* const sums = reinterpret_cast<float*>(lds);                       // [wave][row][kRow]
    float2* const ml = reinterpret_cast<float2*>(sums + NW * 32 * QT * kRow);  // [wave][row]
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int r = wave * 32 * QT + 32 * t + (lane & 31);
        const float l = add_halves(st.l[t]);
        if (half == 0) ml[r] = make_float2(st.m[t] * A.c, l);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x16& o = st.o[t][d];
                *reinterpret_cast<float4*>(sums + r * kRow + 32 * d + 8 * i + 4 * half) =
                    make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            }
    }
    __syncthreads();
    const int here = rows - block * BM < BM ? rows - block * BM : BM;
    for (int i = threadIdx.x; i < here * (DP / 4); i += 64 * NW) {
        const int r = i / (DP / 4), x = i % (DP / 4) * 4;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) top = fmaxf(top, ml[w * 32 * QT + r].x);
        float l = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float2 one = ml[w * 32 * QT + r];
            if (one.y == 0.0f) continue;  // a wave without a visible key (NaN scores leave a NaN sum)
            const float by = exp2_fast(one.x - top);
            const float4 v = *reinterpret_cast<const float4*>(sums + (w * 32 * QT + r) * kRow + x);
            l += one.y * by;
            o.x += v.x * by, o.y += v.y * by, o.z += v.z * by, o.w += v.w * by;
        }
        const int row = D.row + (block * BM + r) / group, head = kvh * group + (block * BM + r) % group;
        const int64_t rh = static_cast<int64_t>(row) * A.heads + head;
        if (parted) {
            *reinterpret_cast<float4*>(A.part_o + (part + rh) * DP + x) = o;
            if (x == 0) A.part_ml[part + rh] = make_float2(top, l);
        } else {
            const float by = l == 0.0f ? 0.0f : 1.0f / l;
            if (x < A.dim) store_four<T>(A.out + row * A.out_row + head * A.out_head + x, o.x * by, o.y * by, o.z * by, o.w * by);
            if (x == 0 && A.lse != nullptr) A.lse[rh] = l == 0.0f ? -INFINITY : top * (1.0f / kLog2E) + logf(l);
        }
    }
}

// The parts of a row and head joined in their order: DP / 4 threads hold a
// row's columns, four each. kMany: all of a workgroup's threads take a row,
// its parts in turn, and their sums meet in LDS (with the parts one after the
// other, a token over 32,000 positions spent 100 of 145 us here). Otherwise
// every DP / 4 threads take a row of their own: fewer, fuller workgroups (8
// trees of 33 tokens over 700-6000 positions, 12 parts: 56 us in all, 65 with
// a workgroup a row; a token over 32,000, 63 parts: 31 and 27 with one). Bound
// by the latency of the sums' reads, 5 to 10 us a call.
template <typename T, int DP, bool kMany>
__global__ __launch_bounds__(256) void tree_join_kernel(const TreeArgs A) {
    constexpr int kCols = DP / 4, kSides = 256 / kCols;
    __shared__ float4 sums[kMany ? kSides : 1][kCols];
    __shared__ float sides_l[kMany ? kSides : 1];
    const int lane = threadIdx.x & 63;
    const int side = threadIdx.x / kCols, col = threadIdx.x % kCols;
    const int64_t all = static_cast<int64_t>(A.n_q) * A.heads;
    const int64_t rh = kMany ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * kSides + side;
    if (rh >= all) return;
    const int row = static_cast<int>(rh / A.heads), head = static_cast<int>(rh % A.heads);
    int lo;
    if (kMany) {
        lo = find_sequence(A.offsets, A.n_seqs, A.n_q, row, lane, [](int, int first) { return first; });
    } else {
        lo = 0;
        for (int hi = A.n_seqs - 1; lo < hi;) {
            const int mid = (lo + hi + 1) / 2;
            if (bounded(A.offsets[mid], A.n_q) <= row) lo = mid; else hi = mid - 1;
        }
    }
    const Drafted D = drafted(A, lo);
    if (row < D.row || row >= D.row + D.n || D.end <= A.chunk) return;
    int parts = (D.end - 1) / A.chunk + 1;
    parts = parts < A.n_splits ? parts : A.n_splits;
    if constexpr (!kMany) {
        join_parts<T, DP>(A.part_o, A.part_ml, all, rh, parts, col, A.dim, A.out + row * A.out_row + head * A.out_head,
                          A.lse != nullptr ? A.lse + rh : nullptr);
        return;
    }
    float top = -INFINITY;
    for (int s = lane; s < parts; s += 64) top = fmaxf(top, A.part_ml[s * all + rh].x);
#pragma unroll
    for (int x = 1; x < 64; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
    float l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s0 = side; s0 < parts; s0 += 4 * kSides) {
        float2 ml[4];
        float4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int s = s0 + i * kSides < parts ? s0 + i * kSides : s0;
            ml[i] = A.part_ml[s * all + rh];
            v[i] = *reinterpret_cast<const float4*>(A.part_o + (s * all + rh) * DP + 4 * col);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (s0 + i * kSides >= parts || ml[i].y == 0.0f) continue;
            const float by = exp2_fast(ml[i].x - top);
            l += ml[i].y * by;
            o.x += v[i].x * by, o.y += v[i].y * by, o.z += v[i].z * by, o.w += v[i].w * by;
        }
    }
    sums[side][col] = o;
    if (col == 0) sides_l[side] = l;
    __syncthreads();
    if (side != 0) return;
    l = 0.0f, o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int i = 0; i < kSides; ++i) {
        const float4 v = sums[i][col];
        l += sides_l[i];
        o.x += v.x, o.y += v.y, o.z += v.z, o.w += v.w;
    }
    const float by = l == 0.0f ? 0.0f : 1.0f / l;
    if (4 * col < A.dim)
        store_four<T>(A.out + row * A.out_row + head * A.out_head + 4 * col, o.x * by, o.y * by, o.z * by, o.w * by);
    if (col == 0 && A.lse != nullptr) A.lse[rh] = l == 0.0f ? -INFINITY : top * (1.0f / kLog2E) + logf(l);
}

// Ancestor bits of drafted tokens: token t's parent is an earlier drafted
// token of its sequence, or any other number where it follows the context. A
// thread walks up from its token, once for each word of its mask: the trees of
// a call are some hundred tokens, one launch's latency.
__global__ __launch_bounds__(256) void tree_masks_kernel(const int32_t* parents, const int32_t* offsets, int n_seqs, int n, int words,
                                                         uint64_t* masks) {
    const int row = blockIdx.x * 256 + threadIdx.x;
    if (row >= n) return;
    int lo = 0, hi = n_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (bounded(offsets[mid], n) <= row) lo = mid; else hi = mid - 1;
    }
    const int first = bounded(offsets[lo], n);
    for (int w = 0; w < words; ++w) {
        uint64_t bits = 0;
        // Parents come before their children, so the walk goes down.
        for (int t = row - first; t >= 0;) {
            if (t >> 6 == w) bits |= uint64_t{1} << (t & 63);
            const int up = parents[first + t];
            t = up < t ? up : -1;
        }
        masks[static_cast<int64_t>(row) * words + w] = bits;
    }
}

constexpr int64_t kMaxPositions = 1 << 30;  // of a sequence, by the checks of its pages
// Keys of a part. At least 512: with 256 two trees of 16 tokens over 20,000
// positions take 55 us, not 47, with 1024 a tree of 64 over 2000 takes 33, not 25.
constexpr int kMinChunk = 512;
// And most of them, so that a long sequence among short ones does not run alone
// (shared tiles, 16 trees over 9000-65000: 340 us, 427 with 8192).
constexpr int kMaxChunk = 8192;
constexpr int kMaxSharedChunk = 4096;
// Of a cache in 8 bits: 16 trees over 9000-65000 313 us, 330 with 4096, 322 with
// 1024. Of 48 shapes (bf16 and fp16, dims 64 to 256, 1 to 48 trees of up to 16 to 64
// tokens over 4000 to 65000 positions) it takes 2% longer than the best of 1024 to
// 8192 on average and 22% at most (dim 64); 1024 5% and 34%, 4096 7% and 61%.
constexpr int kMaxSharedChunk8 = 2048;
constexpr int kSlots = 256;         // workgroups of dealt-out keys that run at a time, one a CU
constexpr int kFewParts = 16;       // at most so many are joined by DP / 4 threads a row
// Workgroups of shared tiles, were all sequences the longest. It sets the keys
// of a part; how many workgroups find rows and keys follows from the lengths (8
// trees over 700-6000 positions: 368 of 1280) and the others return at once.
// Chosen by what calls take: lengths that differ need the parts (16 trees of
// 18-33 tokens over 200-8600 positions: 62 us, 86 with 1024, 116 with 512, 74
// with 2048); trees of one length would do with fewer (6 of 64 tokens over 8000:
// 113 us, 93 with 1024, 125 with 2048), which the host, that knows the longest
// alone, cannot tell apart.
constexpr int kSharedParts = 1280;

// Rows of a workgroup. Up to 32 or 64 rows of a (sequence, head) go to every
// wave and the keys are dealt out to the waves; more rows are dealt out. (32
// trees of 12 tokens, 60 rows, over 3000 positions: 79 us, 106 with the rows
// dealt out; 8 of them 31 and 30. 256 rows a workgroup: 8 trees of up to 33
// tokens 42-58 us, not 36.)
int tree_rows(int dim, int64_t rows) { return rows <= 32 ? 32 : rows <= 64 && dim <= 128 ? 64 : 128; }

// Keys of a part and how many parts the longest sequence has.
void plan_parts(TreeArgs& A, int64_t max_context, bool narrow) {
    const int64_t rows = static_cast<int64_t>(A.max_drafts) * (A.heads / A.kv_heads);
    const int per = tree_rows(A.dim, rows);
    A.row_blocks = static_cast<int32_t>((rows + per - 1) / per);
    // No sequence holds more than 2^30 positions, so a part's first key is an int32.
    const int64_t longest = max_context + A.max_drafts < kMaxPositions ? max_context + A.max_drafts : kMaxPositions;
    const int64_t units = static_cast<int64_t>(A.n_seqs) * A.kv_heads * A.row_blocks;
    int64_t chunk, most = kMaxChunk;
    if (per <= 64) {
        // One round of workgroups: 64 sequences of 2000-8000 positions take
        // 220 us in one part each, 240-260 in two to four.
        chunk = longest / (units > 0 && units < kSlots ? kSlots / units : 1) + 1;
    } else {
        chunk = longest * units / kSharedParts;
        most = narrow ? kMaxSharedChunk8 : kMaxSharedChunk;
    }
    chunk = (chunk + 127) / 128 * 128;
    chunk = chunk < kMinChunk ? kMinChunk : chunk > most ? most : chunk;
    A.chunk = static_cast<int32_t>(chunk);
    A.n_splits = static_cast<int32_t>((longest + chunk - 1) / chunk);
}

template <typename T, int DP, int QT, int NW, bool kShared, bool k8>
int launch_tree_as(TreeArgs& A, hipStream_t s) {
    const int64_t groups = static_cast<int64_t>(A.n_seqs) * A.kv_heads * A.row_blocks * A.n_splits;
    constexpr int KT = kShared && DP <= 128 ? 64 : 32;
    const dim3 grid(static_cast<uint32_t>(groups)), block(64 * NW);
    if (A.page_size % KT == 0)
        hipLaunchKernelGGL((tree_kernel<T, DP, QT, NW, kShared, 2, k8>), grid, block, 0, s, A);
    else if (k8 || A.page_size % Rows<DP>::kPerLoad == 0)  // pages of 8 bits: whole blocks of 16, the rows of a load or several loads'
        hipLaunchKernelGGL((tree_kernel<T, DP, QT, NW, kShared, 1, k8>), grid, block, 0, s, A);
    else if constexpr (!k8)
        hipLaunchKernelGGL((tree_kernel<T, DP, QT, NW, kShared, 0, k8>), grid, block, 0, s, A);
    if (A.n_splits > kFewParts) {
        hipLaunchKernelGGL((tree_join_kernel<T, DP, true>), dim3(static_cast<uint32_t>(A.n_q) * A.heads), dim3(256), 0, s, A);
    } else if (A.n_splits > 1) {
        constexpr int kRows = 1024 / DP;
        hipLaunchKernelGGL((tree_join_kernel<T, DP, false>), dim3((static_cast<uint32_t>(A.n_q) * A.heads + kRows - 1) / kRows), dim3(256), 0, s, A);
    }
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess)
        return fail(AIMG_ERR_HIP, std::string("kernel launch failed: ") + hipGetErrorString(err));
    return AIMG_OK;
}

template <typename T, int DP, bool k8>
int launch_tree(TreeArgs& A, hipStream_t s) {
    const int per = tree_rows(A.dim, static_cast<int64_t>(A.max_drafts) * (A.heads / A.kv_heads));
    if (per == 32) return launch_tree_as<T, DP, 1, DP == 256 ? 2 : 4, false, k8>(A, s);
    if constexpr (DP < 256)
        if (per == 64) return launch_tree_as<T, DP, 2, 4, false, k8>(A, s);
    return launch_tree_as<T, DP, 1, 4, true, k8>(A, s);
}

}  // namespace
}  // namespace aimg

namespace {

// The checks every attention shares: type, element counts, strides that keep
// 16-byte pieces aligned.
// most: of a row's stride.
int check_heads(const aimg_heads* x, const char* name, int64_t most = INT64_MAX, bool written = false) {
    using aimg::fail;
    const std::string n(name);
    if (x == nullptr) return fail(AIMG_ERR_INVALID_ARGUMENT, n + " is null");
    if (x->n_rows < 0 || x->n_rows > INT32_MAX || x->heads < 1 || x->dim < 1)
        return fail(AIMG_ERR_INVALID_ARGUMENT, n + ": n_rows must be in 0..2^31-1, heads and dim at least 1");
    if (x->dim % 8 != 0 || x->dim > aimg::kMaxDim)
        return fail(AIMG_ERR_UNSUPPORTED, n + ": dim must be a multiple of 8 up to " + std::to_string(aimg::kMaxDim) + ", got " + std::to_string(x->dim));
    if (x->n_rows == 0) return AIMG_OK;
    if (x->data == nullptr) return fail(AIMG_ERR_INVALID_ARGUMENT, n + ": null data");
    if (x->row_stride < 0 || x->head_stride < 0) return fail(AIMG_ERR_UNSUPPORTED, n + ": strides must not be negative");
    if (x->row_stride > most && x->n_rows > 1) return fail(AIMG_ERR_UNSUPPORTED, n + ": a row's stride must be at most 2^24 elements");
    const int64_t unit = written ? 4 : 8;
    if (reinterpret_cast<uintptr_t>(x->data) % (2 * unit) != 0 || x->row_stride % unit != 0 || x->head_stride % unit != 0)
        return fail(AIMG_ERR_UNSUPPORTED, n + ": needs a " + std::to_string(2 * unit) + "-byte aligned pointer and strides of whole " +
                                              std::to_string(2 * unit) + " bytes");
    return AIMG_OK;
}

int check_pages(const aimg_pages* p) {
    using aimg::fail;
    if (p == nullptr) return fail(AIMG_ERR_INVALID_ARGUMENT, "pages is null");
    if (p->n_pages < 1 || p->page_size < 1 || p->kv_heads < 1 || p->dim < 1 || p->max_seqs < 1 || p->max_pages < 1)
        return fail(AIMG_ERR_INVALID_ARGUMENT, "pages: every size must be at least 1");
    if (static_cast<int64_t>(p->max_pages) * p->page_size > INT32_MAX / 2)
        return fail(AIMG_ERR_UNSUPPORTED, "pages: a sequence must hold fewer than 2^30 positions");
    if (p->dim % 8 != 0 || p->dim > aimg::kMaxDim)
        return fail(AIMG_ERR_UNSUPPORTED, "pages: dim must be a multiple of 8 up to " + std::to_string(aimg::kMaxDim));
    if (p->k == nullptr || p->v == nullptr || p->page_table == nullptr || p->lengths == nullptr)
        return fail(AIMG_ERR_INVALID_ARGUMENT, "pages: null pointer");
    if ((reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v)) % 16 != 0 || p->page_stride % 8 != 0 ||
        p->slot_stride % 8 != 0 || p->head_stride % 8 != 0 || p->page_stride < 0 || p->head_stride < 0 || p->slot_stride < 0 ||
        p->slot_stride > aimg::kMaxRowStride || p->table_stride < 0)
        return fail(AIMG_ERR_UNSUPPORTED, "pages: needs 16-byte aligned pointers and strides of whole 16 bytes, a position's at most 2^24 elements");
    return AIMG_OK;
}

// What pages of 8-bit elements need besides.
int check_page_scales(const aimg_pages* p, const aimg_page_scales* x) {
    using aimg::fail;
    if (p->dim % 16 != 0) return fail(AIMG_ERR_UNSUPPORTED, "pages: dim must be a multiple of 16 for 8 bits");
    if (p->page_size % aimg::kBlock != 0) return fail(AIMG_ERR_UNSUPPORTED, "pages: page_size must be a multiple of 16 for 8 bits");
    if (p->page_stride % 16 != 0 || p->slot_stride % 16 != 0 || p->head_stride % 16 != 0)
        return fail(AIMG_ERR_UNSUPPORTED, "pages: needs strides of whole 16 bytes");
    if (x->k == nullptr || x->v == nullptr) return fail(AIMG_ERR_INVALID_ARGUMENT, "scales: null pointer");
    if ((reinterpret_cast<uintptr_t>(x->k) | reinterpret_cast<uintptr_t>(x->v)) % 4 != 0 || x->page_stride < 0 || x->head_stride < 0)
        return fail(AIMG_ERR_UNSUPPORTED, "scales: needs 4-byte aligned pointers and strides that are not negative");
    return AIMG_OK;
}

template <typename Launch>
int by_type(int type, int dim, Launch launch) {
    if (type == AIMG_BF16) return launch(aimg::Bf16{}, dim);
    if (type == AIMG_FP16) return launch(aimg::Fp16{}, dim);
    return aimg::fail(AIMG_ERR_UNSUPPORTED, "type must be AIMG_BF16 or AIMG_FP16, got " + std::to_string(type));
}

int check_keys(int64_t n) {
    if (n > aimg::kMostKeys) return aimg::fail(AIMG_ERR_UNSUPPORTED, "prompt attention: needs fewer than 2^31 - 64 rows of keys");
    return AIMG_OK;
}

int check_scale(float scale) {
    if (!(scale > 0.0f) || std::isinf(scale)) return aimg::fail(AIMG_ERR_INVALID_ARGUMENT, "scale must be a positive number");
    return AIMG_OK;
}

}  // namespace

extern "C" int aimg_prompt_workspace_nbytes(int64_t n_rows, int64_t n_keys, int heads, int kv_heads, int dim, int n_seqs,
                                            size_t* nbytes) {
    using aimg::fail;
    if (nbytes == nullptr) return fail(AIMG_ERR_INVALID_ARGUMENT, "nbytes is null");
    if (n_rows < 0 || n_rows > INT32_MAX || n_keys < 0 || n_keys > INT32_MAX || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 ||
        dim < 1 || dim > aimg::kMaxDim || n_seqs < 0)
        return fail(AIMG_ERR_INVALID_ARGUMENT, "prompt attention: rows, keys, heads, dim and n_seqs must be sizes of one call");
    const int rc = check_keys(n_keys);
    if (rc != AIMG_OK) return rc;
    aimg::PromptArgs a{};
    a.n_seqs = n_seqs, a.kv_heads = kv_heads, a.group = heads / kv_heads, a.dim = dim;
    aimg::plan_prompt(a, n_rows, n_keys);
    *nbytes = static_cast<size_t>(a.part_rows) * heads * (4 * aimg::padded_dim(dim) + 8);
    return AIMG_OK;
}

extern "C" int aimg_prompt_attention(const aimg_heads* q, const aimg_heads* k, const aimg_heads* v, const aimg_heads* out,
                                     const int32_t* q_offsets, const int32_t* k_offsets, int n_seqs, int type,
                                     float scale, float* lse, void* workspace, size_t workspace_nbytes, void* stream) {
    using aimg::fail;
    int rc = check_heads(q, "q");
    if (rc == AIMG_OK) rc = check_heads(k, "k", aimg::kMaxRowStride);
    if (rc == AIMG_OK) rc = check_heads(v, "v", aimg::kMaxRowStride);
    if (rc == AIMG_OK) rc = check_heads(out, "out", INT64_MAX, true);
    if (rc == AIMG_OK) rc = check_keys(k->n_rows);
    if (rc == AIMG_OK) rc = check_scale(scale);
    if (rc != AIMG_OK) return rc;
    if (k->n_rows != v->n_rows || k->heads != v->heads || k->dim != q->dim || v->dim != q->dim)
        return fail(AIMG_ERR_INVALID_ARGUMENT, "k and v must have the same rows and heads, and q's dim");
    if (out->n_rows != q->n_rows || out->heads != q->heads || out->dim != q->dim)
        return fail(AIMG_ERR_INVALID_ARGUMENT, "out must have q's shape");
    if (q->heads % k->heads != 0)
        return fail(AIMG_ERR_INVALID_ARGUMENT, "q's heads must be a multiple of k's");
    if (n_seqs < 0) return fail(AIMG_ERR_INVALID_ARGUMENT, "n_seqs must be >= 0");
    if (n_seqs == 0 || q->n_rows == 0) return AIMG_OK;
    if (q_offsets == nullptr || k_offsets == nullptr) return fail(AIMG_ERR_INVALID_ARGUMENT, "null offsets");
    aimg::PromptArgs a{};
    a.q = static_cast<const uint16_t*>(q->data);
    a.k = static_cast<const uint16_t*>(k->data);
    a.v = static_cast<const uint16_t*>(v->data);
    a.out = static_cast<uint16_t*>(out->data);
    a.lse = lse;
    a.q_offsets = q_offsets;
    a.k_offsets = k_offsets;
    a.q_row = q->row_stride, a.q_head = q->head_stride;
    a.k_row = k->row_stride, a.k_head = k->head_stride;
    a.v_row = v->row_stride, a.v_head = v->head_stride;
    a.out_row = out->row_stride, a.out_head = out->head_stride;
    a.n_seqs = n_seqs, a.heads = q->heads, a.kv_heads = k->heads, a.group = q->heads / k->heads, a.dim = q->dim;
    a.n_q = static_cast<int32_t>(q->n_rows), a.n_k = static_cast<int32_t>(k->n_rows);
    a.c = scale * aimg::kLog2E, a.scale = scale;
    aimg::plan_prompt(a, q->n_rows, k->n_rows);
    const int64_t part_rows = static_cast<int64_t>(a.part_rows) * q->heads;
    const int dp = aimg::padded_dim(q->dim);
    if (a.n_splits > 1 && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 ||
                           workspace_nbytes < static_cast<size_t>(part_rows) * (4 * dp + 8)))
        return fail(AIMG_ERR_INVALID_ARGUMENT, "the workspace is null, misaligned or below aimg_prompt_workspace_nbytes");
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + part_rows * dp);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return by_type(type, q->dim, [&](auto t, int dim) {
        typedef decltype(t) T;
        if (dim <= 64) return aimg::launch_prompt<T, 64>(a, s);
        if (dim <= 128) return aimg::launch_prompt<T, 128>(a, s);
        return aimg::launch_prompt<T, 256>(a, s);
    });
}

namespace {

// What the sizes of one tree attention call imply.
int tree_sizes(aimg::TreeArgs& a, int64_t n_rows, int n_seqs, int heads, int kv_heads, int dim, int max_drafts, int64_t max_context,
               bool narrow) {
    using aimg::fail;
    if (n_rows < 0 || n_rows > INT32_MAX || n_seqs < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || dim < 1 ||
        dim > aimg::kMaxDim || max_drafts < 1 || max_context < 0 || max_context > INT32_MAX)
        return fail(AIMG_ERR_INVALID_ARGUMENT, "tree attention: n_seqs and max_context must be >= 0 (max_context below 2^31), max_drafts >= 1, "
                                               "rows, heads and dim sizes of one call");
    if (n_rows * heads > INT32_MAX) return fail(AIMG_ERR_UNSUPPORTED, "tree attention: too many rows times heads");
    a.n_seqs = n_seqs, a.heads = heads, a.kv_heads = kv_heads, a.dim = dim;
    a.max_drafts = max_drafts < n_rows ? max_drafts : n_rows > 0 ? static_cast<int32_t>(n_rows) : 1;  // no sequence has more
    const int64_t blocks = (static_cast<int64_t>(a.max_drafts) * (heads / kv_heads) + 31) / 32;  // at least the row blocks
    if (static_cast<int64_t>(n_seqs) * kv_heads > INT32_MAX / blocks)
        return fail(AIMG_ERR_UNSUPPORTED, "tree attention: too many sequences, heads and rows");
    aimg::plan_parts(a, max_context, narrow);
    if (static_cast<int64_t>(n_seqs) * kv_heads * a.row_blocks > INT32_MAX / a.n_splits)
        return fail(AIMG_ERR_UNSUPPORTED, "tree attention: too many sequences, heads and keys");
    return AIMG_OK;
}

int tree_workspace(int64_t n_rows, int heads, int kv_heads, int dim, int n_seqs, int max_drafts, int64_t max_context, bool narrow,
                   size_t* nbytes) {
    using aimg::fail;
    if (nbytes == nullptr) return fail(AIMG_ERR_INVALID_ARGUMENT, "nbytes is null");
    aimg::TreeArgs a{};
    const int rc = tree_sizes(a, n_rows, n_seqs, heads, kv_heads, dim, max_drafts, max_context, narrow);
    if (rc != AIMG_OK) return rc;
    const int64_t rows = n_rows * heads * a.n_splits;
    *nbytes = a.n_splits > 1 ? static_cast<size_t>(rows) * (4 * aimg::padded_dim(dim) + 8) : 0;
    return AIMG_OK;
}

}  // namespace

extern "C" int aimg_tree_workspace_nbytes(int64_t n_rows, int heads, int kv_heads, int dim, int n_seqs, int max_drafts,
                                          int64_t max_context, size_t* nbytes) {
    return tree_workspace(n_rows, heads, kv_heads, dim, n_seqs, max_drafts, max_context, false, nbytes);
}

extern "C" int aimg_tree8_workspace_nbytes(int64_t n_rows, int heads, int kv_heads, int dim, int n_seqs, int max_drafts,
                                           int64_t max_context, size_t* nbytes) {
    return tree_workspace(n_rows, heads, kv_heads, dim, n_seqs, max_drafts, max_context, true, nbytes);
}

namespace {

// Over a cache in 16 bits (scales null) or 8.
int tree_attention(const aimg_heads* q, const aimg_pages* pages, const aimg_page_scales* scales, const aimg_heads* out,
                   const int32_t* seqs, const int32_t* draft_offsets, int n_seqs, const int64_t* masks, int mask_words, int max_drafts,
                   int64_t max_context, int type, float scale, float* lse, void* workspace, size_t workspace_nbytes, void* stream) {
    using aimg::fail;
    int rc = check_heads(q, "q");
    if (rc == AIMG_OK) rc = check_heads(out, "out", INT64_MAX, true);
    if (rc == AIMG_OK) rc = check_pages(pages);
    if (rc == AIMG_OK && scales != nullptr) rc = check_page_scales(pages, scales);
    if (rc == AIMG_OK) rc = check_scale(scale);
    if (rc != AIMG_OK) return rc;
    if (out->n_rows != q->n_rows || out->heads != q->heads || out->dim != q->dim)
        return fail(AIMG_ERR_INVALID_ARGUMENT, "out must have q's shape");
    if (q->dim != pages->dim || q->heads % pages->kv_heads != 0)
        return fail(AIMG_ERR_INVALID_ARGUMENT, "q must have the pages' dim and a multiple of their heads");
    aimg::TreeArgs a{};
    rc = tree_sizes(a, q->n_rows, n_seqs, q->heads, pages->kv_heads, q->dim, max_drafts, max_context, scales != nullptr);
    if (rc != AIMG_OK) return rc;
    if (masks != nullptr && mask_words < 1) return fail(AIMG_ERR_INVALID_ARGUMENT, "mask_words must be >= 1");
    if (n_seqs == 0 || q->n_rows == 0) return AIMG_OK;
    if (seqs == nullptr || draft_offsets == nullptr) return fail(AIMG_ERR_INVALID_ARGUMENT, "null seqs or draft_offsets");
    if (scales != nullptr)
        a.k_scales = scales->k, a.v_scales = scales->v, a.scale_page = scales->page_stride, a.scale_head = scales->head_stride;
    const int64_t part_rows = q->n_rows * q->heads * a.n_splits;
    const int dp = aimg::padded_dim(q->dim);
    if (a.n_splits > 1 && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 ||
                           workspace_nbytes < static_cast<size_t>(part_rows) * (4 * dp + 8)))
        return fail(AIMG_ERR_INVALID_ARGUMENT, "the workspace is null, misaligned or below aimg_tree_workspace_nbytes");
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + part_rows * dp);
    a.q = static_cast<const uint16_t*>(q->data);
    a.k = static_cast<const char*>(pages->k);
    a.v = static_cast<const char*>(pages->v);
    a.out = static_cast<uint16_t*>(out->data);
    a.lse = lse;
    a.table = pages->page_table, a.lengths = pages->lengths, a.seqs = seqs, a.offsets = draft_offsets;
    a.masks = reinterpret_cast<const uint64_t*>(masks);
    a.words = mask_words;
    a.q_row = q->row_stride, a.q_head = q->head_stride;
    a.out_row = out->row_stride, a.out_head = out->head_stride;
    a.page_stride = pages->page_stride, a.slot_stride = pages->slot_stride, a.kv_head_stride = pages->head_stride;
    a.table_stride = pages->table_stride, a.max_pages = pages->max_pages, a.n_slots = pages->max_seqs;
    a.n_pages = pages->n_pages, a.page_size = pages->page_size;
    a.n_q = static_cast<int32_t>(q->n_rows);
    a.magic = pages->page_size == 1 ? 0xFFFFFFFFu : static_cast<uint32_t>((uint64_t{1} << 32) / pages->page_size);
    a.c = scale * aimg::kLog2E, a.scale = scale;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return by_type(type, q->dim, [&](auto t, int dim) {
        typedef decltype(t) T;
        if (scales != nullptr) {
            if (dim <= 64) return aimg::launch_tree<T, 64, true>(a, s);
            if (dim <= 128) return aimg::launch_tree<T, 128, true>(a, s);
            return aimg::launch_tree<T, 256, true>(a, s);
        }
        if (dim <= 64) return aimg::launch_tree<T, 64, false>(a, s);
        if (dim <= 128) return aimg::launch_tree<T, 128, false>(a, s);
        return aimg::launch_tree<T, 256, false>(a, s);
    });
}

}  // namespace

extern "C" int aimg_tree_attention(const aimg_heads* q, const aimg_pages* pages, const aimg_heads* out, const int32_t* seqs,
                                   const int32_t* draft_offsets, int n_seqs, const int64_t* masks, int mask_words, int max_drafts,
                                   int64_t max_context, int type, float scale, float* lse, void* workspace,
                                   size_t workspace_nbytes, void* stream) {
    return tree_attention(q, pages, nullptr, out, seqs, draft_offsets, n_seqs, masks, mask_words, max_drafts, max_context, type, scale,
                          lse, workspace, workspace_nbytes, stream);
}

extern "C" int aimg_tree8_attention(const aimg_heads* q, const aimg_pages* pages, const aimg_page_scales* scales, const aimg_heads* out,
                                    const int32_t* seqs, const int32_t* draft_offsets, int n_seqs, const int64_t* masks, int mask_words,
                                    int max_drafts, int64_t max_context, int type, float scale, float* lse, void* workspace,
                                    size_t workspace_nbytes, void* stream) {
    if (scales == nullptr) return aimg::fail(AIMG_ERR_INVALID_ARGUMENT, "scales is null");
    return tree_attention(q, pages, scales, out, seqs, draft_offsets, n_seqs, masks, mask_words, max_drafts, max_context, type, scale, lse,
                          workspace, workspace_nbytes, stream);
}


extern "C" int aimg_tree_masks(const int32_t* parents, const int32_t* draft_offsets, int n_seqs, int64_t n_rows, int mask_words,
                               int64_t* masks, void* stream) {
    using aimg::fail;
    if (n_seqs < 0 || n_rows < 0 || n_rows > INT32_MAX || mask_words < 1)
        return fail(AIMG_ERR_INVALID_ARGUMENT, "n_seqs and n_rows must be >= 0 (n_rows below 2^31) and mask_words >= 1");
    if (n_seqs == 0 || n_rows == 0) return AIMG_OK;
    if (parents == nullptr || draft_offsets == nullptr || masks == nullptr)
        return fail(AIMG_ERR_INVALID_ARGUMENT, "null pointer passed to aimg_tree_masks");
    hipLaunchKernelGGL(aimg::tree_masks_kernel, dim3(static_cast<uint32_t>((n_rows + 255) / 256)), dim3(256), 0,
                       static_cast<hipStream_t>(stream), parents, draft_offsets, n_seqs, static_cast<int>(n_rows), mask_words,
                       reinterpret_cast<uint64_t*>(masks));
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess)
        return fail(AIMG_ERR_HIP, std::string("kernel launch failed: ") + hipGetErrorString(err));
    return AIMG_OK;
}
