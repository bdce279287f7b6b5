// paged_attend.hpp — the arithmetic that the paged attention kernels share: a
// tile of cached rows in registers, the query as a matrix operand, a softmax
// with a running maximum, and the products of the three (paged_attention.hip
// gives the layout).
#pragma once

#include "device.hpp"
#include "paged_device.hpp"

namespace nut {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <int TYPE>
__device__ __forceinline__ f32x4 product(u32x4 a, u32x4 b, f32x4 c)
{
    if constexpr (TYPE == NUT_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// The limbs of eight finite fp32 values as matrix operands.
template <int TYPE, int LIMBS>
__device__ __forceinline__ void split(const float (&x)[8], u32x4 (&limb)[LIMBS])
{
#pragma unroll
    for (int w = 0; w < 4; w++) {
        float a = x[2 * w], b = x[2 * w + 1];
#pragma unroll
        for (int l = 0; l < LIMBS; l++) {
            if constexpr (TYPE == NUT_BF16) {
                // the upper half of the bits: what is cut off is the rest, exactly
                const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
                limb[l][w] = __builtin_amdgcn_perm(ub, ua, 0x07060302);
                a -= __uint_as_float(ua & 0xffff0000u);
                b -= __uint_as_float(ub & 0xffff0000u);
            } else {
                const uint32_t ha = to_f16(a), hb = to_f16(b);
                limb[l][w] = ha | (hb << 16);
                a -= from_f16(ha);
                b -= from_f16(hb);
            }
        }
    }
}

__device__ __forceinline__ float max_over_rows(float v)
{
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// One wave's softmax over the tiles it has seen, for the head of its lane:
// weights are 2^(score - ref), ref = most - 14 for fp16 rows and most else
// (0 before the first score that is not minus infinity).
template <int TYPE, int HD> struct Softmax {
    static constexpr int G = HD / 16;
    static constexpr float kShift = TYPE == NUT_F16 ? 14.0f : 0.0f;
    float most = -INFINITY, ref = 0.0f, sum = 0.0f;
    f32x4 o[G];

    __device__ __forceinline__ Softmax()
    {
#pragma unroll
        for (int t = 0; t < G; t++)
            o[t] = f32x4{0, 0, 0, 0};
    }
    // Raises the running maximum; what was summed is scaled to it.
    __device__ __forceinline__ void raise(float tile)
    {
        const float now = fmaxf(most, tile);
        if (__any(now > most)) {
            const float to = now == -INFINITY ? 0.0f : now - kShift;
            const float f = most == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ref - to);
            // a sum that is not a number stays one
            sum = most == -INFINITY ? sum : sum * f;
#pragma unroll
            for (int t = 0; t < G; t++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    o[t][i] = most == -INFINITY ? o[t][i] : o[t][i] * f;
            most = now, ref = to;
        }
    }
};

// The rows of one tile in registers: 32 rows of 16 bits or 16 of 32.
template <int TYPE, int HD> struct Tile {
    static constexpr int G = HD / 16;
    static constexpr bool kWide = TYPE == NUT_F32;
    static constexpr int kRows = kWide ? 16 : 32;
    static constexpr int kScores = kRows / 4;            // of a lane
    static constexpr int kKeys = HD / 16;                // 16-byte pieces of K
    static constexpr int kWords = kWide ? G : G / 2;     // of a V row
    // pieces of a power of two words divide a row of 8 n components
    static constexpr int kPiece = kWords % 4 == 0 ? 4 : kWords % 2 == 0 ? 2 : 1;
    static constexpr int kEach = kWide ? kPiece : 2 * kPiece; // components of a piece
    u32x4 k[kKeys];
    uint32_t v[kScores][kWords];

    // Component t of the lane's eight 16-bit rows, as a matrix operand.
    __device__ __forceinline__ u32x4 component(int t) const
    {
        u32x4 x;
#pragma unroll
        for (int w = 0; w < 4; w++)
            x[w] = __builtin_amdgcn_perm(v[2 * w + 1][t / 2], v[2 * w][t / 2],
                                         t % 2 ? 0x07060302 : 0x05040100);
        return x;
    }
    template <bool NT, typename V> static __device__ __forceinline__ V fetch(const char *p)
    {
        const V *q = reinterpret_cast<const V *>(p);
        return NT ? __builtin_nontemporal_load(q) : *q;
    }
    // FULL: the head dim is HD; else components beyond it count zero. NT: past
    // the caches' replacement.
    template <bool FULL, bool NT>
    __device__ __forceinline__ void load(const PagedView &kv, const size_t *at, int lane)
    {
        const int j = lane >> 4, c = lane & 15;
        constexpr int kSize = kWide ? 4 : 2;
        constexpr int kParts = kWide ? HD / 16 : HD / 32; // pieces of a row's 16 j .. 16 j + 15
#pragma unroll
        for (int sub = 0; sub < kRows / 16; sub++) {
            const char *p = kv.keys + at[16 * sub + c];
#pragma unroll
            for (int n = 0; n < kParts; n++) {
                const uint32_t byte = n * 64 + j * 16;
                const bool in = FULL || byte < kv.head_dim * kSize;
                u32x4 x{0, 0, 0, 0};
                if (in)
                    x = fetch<NT, u32x4>(p + byte);
                k[sub * kParts + n] = x;
            }
        }
#pragma unroll
        for (int r = 0; r < kScores; r++) {
            const char *p = kv.values + at[16 * (r / 4) + 4 * j + r % 4];
#pragma unroll
            for (int w = 0; w < kWords; w += kPiece) {
                const uint32_t byte = (16 * w + c * kPiece) * 4;
                const char *q = p + (FULL || byte < kv.head_dim * kSize ? byte : 0);
                if constexpr (kPiece == 1) {
                    v[r][w] = fetch<NT, uint32_t>(q);
                } else if constexpr (kPiece == 2) {
                    const u32x2 x = fetch<NT, u32x2>(q);
                    v[r][w] = x[0], v[r][w + 1] = x[1];
                } else {
                    const u32x4 x = fetch<NT, u32x4>(q);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        v[r][w + e] = x[e];
                }
            }
        }
    }
};

// The query of the lane's head as a matrix operand, scaled to base 2.
template <int TYPE, int HD> struct Query {
    static constexpr int kLimbs = TYPE == NUT_F32 ? 1 : TYPE == NUT_F16 ? 2 : 3;
    static constexpr int kParts = TYPE == NUT_F32 ? HD / 16 : HD / 32;
    static constexpr int kEach = TYPE == NUT_F32 ? 4 : 8;
    float v[kParts][kEach]; // as it was read
    u32x4 x[kParts][kLimbs];
    int exponent = 0; // scores come out divided by 2^exponent

    __device__ __forceinline__ void fetch(const float *q, bool valid, uint32_t head_dim, int lane)
    {
        const int j = lane >> 4;
#pragma unroll
        for (int n = 0; n < kParts; n++) {
            const uint32_t d = n * 4 * kEach + j * kEach;
#pragma unroll
            for (int e = 0; e < kEach; e += 4) {
                float4 f = make_float4(0, 0, 0, 0);
                if (valid && d + e < head_dim)
                    f = *reinterpret_cast<const float4 *>(q + d + e);
                v[n][e] = f.x, v[n][e + 1] = f.y, v[n][e + 2] = f.z, v[n][e + 3] = f.w;
            }
        }
    }
    __device__ __forceinline__ void convert(float scale)
    {
        float most = 0.0f, odd = 0.0f;
#pragma unroll
        for (int n = 0; n < kParts; n++)
#pragma unroll
            for (int e = 0; e < kEach; e++) {
                v[n][e] *= scale;
                most = fmaxf(most, fabsf(v[n][e]));
                odd = fmaf(v[n][e], 0.0f, odd); // not a number after one that is not finite
            }
        if constexpr (TYPE == NUT_F32) {
#pragma unroll
            for (int n = 0; n < kParts; n++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    x[n][0][e] = __float_as_uint(v[n][e]);
        } else {
            if constexpr (TYPE == NUT_F16) {
                if (__any(most == INFINITY)) { // the finite ones have to fit limbs all the same
                    most = 0.0f;
#pragma unroll
                    for (int n = 0; n < kParts; n++)
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            most = fabsf(v[n][e]) < INFINITY ? fmaxf(most, fabsf(v[n][e])) : most;
                }
                most = max_over_rows(most);
                if (most > 0.0f)
                    exponent = ilogbf(most) - 13;
#pragma unroll
                for (int n = 0; n < kParts; n++)
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        v[n][e] = ldexpf(v[n][e], -exponent);
            }
            const bool rare = __any(odd != odd);
            if (rare) { // cut to its upper half, a NaN may look infinite
#pragma unroll
                for (int n = 0; n < kParts; n++)
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        v[n][e] = v[n][e] != v[n][e] ? __uint_as_float(0x7fc00000u) : v[n][e];
            }
#pragma unroll
            for (int n = 0; n < kParts; n++)
                split<TYPE, kLimbs>(v[n], x[n]);
            if (rare) { // inf - inf is not a limb
#pragma unroll
                for (int n = 0; n < kParts; n++)
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        const uint32_t lo = fabsf(v[n][2 * w]) < INFINITY ? 0xffffu : 0;
                        const uint32_t hi = fabsf(v[n][2 * w + 1]) < INFINITY ? 0xffff0000u : 0;
#pragma unroll
                        for (int l = 1; l < kLimbs; l++)
                            x[n][l][w] &= lo | hi;
                    }
            }
        }
    }
};

// The scores of a tile's rows for the head of the lane, base 2: of rows
// 4 j + i (lane = 16 j + c), then, of 16-bit rows, 16 + 4 j + i.
template <int TYPE, int HD>
__device__ __forceinline__ void score(const Tile<TYPE, HD> &tile, const Query<TYPE, HD> &q,
                                      float (&s)[Tile<TYPE, HD>::kScores])
{
    using T = Tile<TYPE, HD>;
    if constexpr (T::kWide) {
        f32x4 acc{0, 0, 0, 0};
#pragma unroll
        for (int n = 0; n < T::kKeys; n++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(tile.k[n][e]),
                                                           __uint_as_float(q.x[n][0][e]), acc, 0,
                                                           0, 0);
#pragma unroll
        for (int i = 0; i < 4; i++)
            s[i] = acc[i];
    } else {
        constexpr int kParts = HD / 32;
#pragma unroll
        for (int sub = 0; sub < 2; sub++) {
            f32x4 acc{0, 0, 0, 0};
#pragma unroll
            for (int n = 0; n < kParts; n++)
#pragma unroll
                for (int l = Query<TYPE, HD>::kLimbs - 1; l >= 0; l--)
                    acc = product<TYPE>(tile.k[sub * kParts + n], q.x[n][l], acc);
            const bool odd = acc[0] + acc[1] + acc[2] + acc[3] != acc[0] + acc[1] + acc[2] + acc[3];
            if (__any(odd)) {
                // An infinite key: the first limb's product has the sum's sign, a
                // later limb of zero, or of the other sign, makes it no number.
                f32x4 first{0, 0, 0, 0};
#pragma unroll
                for (int n = 0; n < kParts; n++)
                    first = product<TYPE>(tile.k[sub * kParts + n], q.x[n][0], first);
#pragma unroll
                for (int i = 0; i < 4; i++)
                    acc[i] = acc[i] != acc[i] ? first[i] : acc[i];
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
                s[4 * sub + i] = TYPE == NUT_F16 ? ldexpf(acc[i], q.exponent) : acc[i];
        }
    }
}

// `gone`: bit r set where row r of the tile is masked, the same in every lane.
template <int TYPE, int HD>
__device__ __forceinline__ void attend(Tile<TYPE, HD> &tile, uint32_t gone,
                                       const Query<TYPE, HD> &q, Softmax<TYPE, HD> &sm,
                                       float *scores, int lane)
{
    using T = Tile<TYPE, HD>;
    constexpr int G = T::G;
    float s[T::kScores];
    score<TYPE, HD>(tile, q, s);
    if (gone != 0) { // a masked row may hold NaN, and 0 NaN is NaN
        const uint32_t mine = gone >> (4 * (lane >> 4));
#pragma unroll
        for (int r = 0; r < T::kScores; r++) {
            const bool out = mine >> (16 * (r / 4) + r % 4) & 1;
            s[r] = out ? -INFINITY : s[r];
#pragma unroll
            for (int w = 0; w < T::kWords; w++)
                tile.v[r][w] = out ? 0 : tile.v[r][w];
        }
    }
    if (scores != nullptr) {
#pragma unroll
        for (int sub = 0; sub < T::kRows / 16; sub++)
            *reinterpret_cast<float4 *>(scores + 16 * sub) =
                make_float4(s[4 * sub], s[4 * sub + 1], s[4 * sub + 2], s[4 * sub + 3]);
    }
    float most = s[0];
#pragma unroll
    for (int r = 1; r < T::kScores; r++)
        most = fmaxf(most, s[r]);
    sm.raise(max_over_rows(most));
    float p[8];
#pragma unroll
    for (int r = 0; r < T::kScores; r++) {
        p[r] = __builtin_amdgcn_exp2f(s[r] - sm.ref);
        sm.sum += p[r];
    }
    const auto &v = tile.v;
    if constexpr (T::kWide) {
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int t = 0; t < G; t++)
                sm.o[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[r][t]), p[r],
                                                               sm.o[t], 0, 0, 0);
    } else {
        constexpr int kLimbs = Query<TYPE, HD>::kLimbs;
        u32x4 limb[kLimbs];
        split<TYPE, kLimbs>(p, limb);
#pragma unroll
        for (int t = 0; t < G; t++) {
            const u32x4 x = tile.component(t);
#pragma unroll
            for (int l = kLimbs - 1; l >= 0; l--)
                sm.o[t] = product<TYPE>(x, limb[l], sm.o[t]);
        }
    }
}

} // namespace nut
