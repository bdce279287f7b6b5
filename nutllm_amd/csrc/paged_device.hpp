// paged_device.hpp — device helpers of the paged KV cache kernels.
#pragma once

#include "paged.hpp"

namespace nut {

__device__ __forceinline__ void paged_flag(int *status, int bit)
{
    if (status != nullptr)
        atomicOr(status, bit);
}

// Rows of sequence b; 0, flagged once by the caller's `report` thread, where
// the length is not one that the call allows.
__device__ __forceinline__ uint32_t paged_length(const PagedView &kv, const PagedSeqs &s,
                                                 uint32_t b, bool report)
{
    const int n = s.lengths[b];
    if (length_in(n, s.max_length))
        return uint32_t(n);
    if (report)
        paged_flag(kv.status, kBadLength);
    return 0;
}

constexpr size_t kNoRow = ~size_t(0);

// Byte offset of `slot` of the sequence's page `index`, for KV head h;
// kNoRow, flagged, where the table names no page of the cache.
__device__ __forceinline__ size_t paged_row(const PagedView &kv, const PagedSeqs &s, uint32_t b,
                                            uint32_t index, uint32_t slot, uint32_t h)
{
    const int page = s.table[size_t(b) * s.table_stride + index];
    if (!page_in(page, kv.pages)) {
        paged_flag(kv.status, kBadPage);
        return kNoRow;
    }
    return size_t(page) * kv.page_stride + size_t(h) * kv.head_stride +
           size_t(slot) * kv.slot_stride;
}

__device__ __forceinline__ float from_bf16(uint32_t bits)
{
    return __uint_as_float(bits << 16);
}

__device__ __forceinline__ float from_f16(uint32_t bits)
{
    return float(__builtin_bit_cast(_Float16, uint16_t(bits)));
}

// fp32 to bfloat16, to nearest, ties to even; a NaN stays one.
__device__ __forceinline__ uint32_t to_bf16(float v)
{
    const uint32_t u = __float_as_uint(v);
    if ((u & 0x7fffffffu) > 0x7f800000u)
        return (u >> 16) | 0x40u;
    return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}

__device__ __forceinline__ uint32_t to_f16(float v)
{
    return __builtin_bit_cast(uint16_t, _Float16(v));
}

// Eight consecutive components of a row, 16-byte aligned.
template <int TYPE> __device__ __forceinline__ void load8(const char *p, float (&v)[8])
{
    if constexpr (TYPE == NUT_F32) {
        const float4 a = reinterpret_cast<const float4 *>(p)[0];
        const float4 b = reinterpret_cast<const float4 *>(p)[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
        v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const uint4 u = *reinterpret_cast<const uint4 *>(p);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i] = TYPE == NUT_BF16 ? from_bf16(w[i] & 0xffffu) : from_f16(w[i] & 0xffffu);
            v[2 * i + 1] = TYPE == NUT_BF16 ? from_bf16(w[i] >> 16) : from_f16(w[i] >> 16);
        }
    }
}

// Rounds eight components to TYPE in place and stores them.
template <int TYPE> __device__ __forceinline__ void store8(char *p, float (&v)[8])
{
    if constexpr (TYPE == NUT_F32) {
        reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t bits = TYPE == NUT_BF16 ? to_bf16(v[i]) : to_f16(v[i]);
            v[i] = TYPE == NUT_BF16 ? from_bf16(bits) : from_f16(bits);
            w[i / 2] = i % 2 == 0 ? bits : w[i / 2] | (bits << 16);
        }
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// The smaller and the larger of two values; a NaN wins, so that a page's
// bounds show it.
__device__ __forceinline__ float lower(float a, float b) { return b < a || b != b ? b : a; }
__device__ __forceinline__ float upper(float a, float b) { return b > a || b != b ? b : a; }

} // namespace nut
