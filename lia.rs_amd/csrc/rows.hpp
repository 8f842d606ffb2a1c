// Rows of keys and values on their way into and out of a paged KV pool (gfx950): slots, source and pool elements by eights.
#pragma once

#include "common.hpp"

namespace lia {

// The kernels' number of a source or output type, -1 for others.
inline int src_kind_of(int32_t dtype) {
    return dtype == LIA_F32 ? 0 : dtype == LIA_F16 ? 1 : dtype == LIA_BF16 ? 2 : -1;
}

// FP8 page scale for an append.  A page appended to before it was ever quantised holds
// scale 0; it takes scale 1, which the appending threads record (every writer stores the
// same value, and readers after the append see 1).
__device__ __forceinline__ float append_scale(float *scales, size_t at) {
    float s = scales[at];
    if (s == 0.0f) {
        s = 1.0f;
        scales[at] = 1.0f;
    }
    return s;
}

// Slot of append row r (slot_mapping[r], or the table's page of its position); kNone for
// "no slot", for a position past its table row, whose page another sequence may own, and for any
// slot outside the pool: such a row is not written.
__device__ __forceinline__ uint32_t row_slot(uint32_t r, const uint32_t *slot_mapping,
                                             const uint32_t *positions, const uint32_t *sequences,
                                             const uint32_t *pages, uint32_t stride,
                                             uint32_t page_shift, uint32_t pool_pages) {
    if (slot_mapping) {
        const uint32_t slot = slot_mapping[r];
        return (slot >> page_shift) < pool_pages ? slot : kNone;
    }
    const uint32_t pos = positions[r];
    if ((pos >> page_shift) >= stride) return kNone;
    const uint32_t page = pages[(size_t)sequences[r] * stride + (pos >> page_shift)];
    return page < pool_pages ? page * (1u << page_shift) + (pos & ((1u << page_shift) - 1)) : kNone;
}

// Eight consecutive source elements from index i (a multiple of 8 of a 16-byte aligned array) as
// f32.  SRC: 0 = f32, 1 = f16, 2 = bf16.
template <int SRC>
__device__ __forceinline__ void load8(const void *p, size_t i, float (&x)[8]) {
    if constexpr (SRC == 0) {
        const float4 a = ((const float4 *)p)[i / 4], b = ((const float4 *)p)[i / 4 + 1];
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
        const u32x4 w = ((const u32x4 *)p)[i / 8];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            x[2 * j] = SRC == 1 ? f16_to_f32(w[j] & 0xffffu) : bf16_to_f32(w[j] & 0xffffu);
            x[2 * j + 1] = SRC == 1 ? f16_to_f32(w[j] >> 16) : bf16_to_f32(w[j] >> 16);
        }
    }
}

// Eight consecutive pool elements (16 or, FP8, 8 bytes, aligned to their size).
template <int KVT>
__device__ __forceinline__ void store8(void *pool, size_t at, const float (&x)[8], const Divisor &d) {
    if constexpr (KVT == LIA_FP8_E4M3) {
        float q[8];
#pragma unroll
        for (int j = 0; j < 8; j++) q[j] = quotient(x[j], d);
        *(u32x2 *)((uint8_t *)pool + at) = u32x2{f32x4_to_e4m3x4(q[0], q[1], q[2], q[3]),
                                                 f32x4_to_e4m3x4(q[4], q[5], q[6], q[7])};
    } else {
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t lo = KVT == LIA_BF16 ? f32_to_bf16(x[2 * j]) : f32_to_f16(x[2 * j]);
            const uint32_t hi = KVT == LIA_BF16 ? f32_to_bf16(x[2 * j + 1]) : f32_to_f16(x[2 * j + 1]);
            w[j] = lo | (hi << 16);
        }
        *(u32x4 *)((uint16_t *)pool + at) = w;
    }
}

// Largest magnitude (as bits) over the N lanes of an aligned group.
template <int N>
__device__ __forceinline__ uint32_t group_max(uint32_t x) {
#pragma unroll
    for (int o = 1; o < N; o <<= 1) x = max(x, (uint32_t)__shfl_xor((int)x, o));
    return x;
}

// First code byte / 16 of the block that holds element e of KV head h of `slot` in an MXFP4 pool.
__device__ __forceinline__ size_t mxfp4_block(uint32_t slot, uint32_t page_shift, uint32_t hkv, uint32_t h,
                                              uint32_t hd, uint32_t e) {
    const uint32_t page = slot >> page_shift, off = slot & ((1u << page_shift) - 1);
    return ((((size_t)page * hkv + h) << page_shift) + off) * (hd / 32) + e / 32;
}

// Eight elements (piece e8 of their head's) of one MXFP4 block held by four neighbouring lanes: its scale over the lanes, this
// lane's four code bytes, the scale by the block's first lane.
__device__ __forceinline__ void store8_fp4(uint8_t *codes, uint8_t *scales, size_t block, uint32_t e8,
                                           const float (&x)[8]) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) top = max(top, f2u(x[j]) & 0x7fffffffu);
    const uint32_t s = mxfp4_scale(group_max<4>(top));
    const float inv = mxfp4_inverse(s);
    uint32_t w = 0; // a NaN block's codes
    if (s != 255)
        w = f32x4_to_e2m1x4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv) |
            f32x4_to_e2m1x4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv) << 16;
    ((uint32_t *)codes)[block * 4 + (e8 & 3)] = w;
    if ((e8 & 3) == 0) scales[block] = (uint8_t)s;
}

// Eight consecutive elements from e of KV head h of the pool row `slot`, as f32.
template <int KVT>
__device__ __forceinline__ void values8(const void *pool, const void *scales, uint32_t slot, uint32_t page_shift,
                                        uint32_t hkv, uint32_t h, uint32_t hd, uint32_t e, float (&x)[8]) {
    const size_t at = ((size_t)slot * hkv + h) * hd + e;
    if constexpr (KVT == LIA_FP4) {
        const size_t b = mxfp4_block(slot, page_shift, hkv, h, hd, e);
        const uint32_t w = ((const uint32_t *)pool)[b * 4 + (e & 31) / 8];
        const u32x4 y = e2m1x8_to_bf16x8(w, u2f((uint32_t)((const uint8_t *)scales)[b] << 23));
#pragma unroll
        for (int j = 0; j < 4; j++) {
            x[2 * j] = bf16_to_f32(y[j] & 0xffffu);
            x[2 * j + 1] = bf16_to_f32(y[j] >> 16);
        }
    } else if constexpr (KVT == LIA_FP8_E4M3) {
        const u32x2 w = *(const u32x2 *)((const uint8_t *)pool + at);
        const float s = ((const float *)scales)[(size_t)(slot >> page_shift) * hkv + h];
        const u32x4 y = e4m3x8_to_f16x8(w);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            x[2 * j] = f16_to_f32(y[j] & 0xffffu) * s;
            x[2 * j + 1] = f16_to_f32(y[j] >> 16) * s;
        }
    } else {
        load8<KVT == LIA_F16 ? 1 : 2>(pool, at, x);
    }
}

template <int DST>
__device__ __forceinline__ void put8(void *out, size_t i, const float (&x)[8]) {
    if constexpr (DST == 0) {
        ((float4 *)out)[i / 4] = make_float4(x[0], x[1], x[2], x[3]);
        ((float4 *)out)[i / 4 + 1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        store8<DST == 1 ? LIA_F16 : LIA_BF16>(out, i, x, Divisor{});
    }
}

} // namespace lia
