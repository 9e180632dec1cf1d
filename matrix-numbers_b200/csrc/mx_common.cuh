// Microscaled (MX) operands: element formats, the block scale and the layout that the MX kernels share.
//
// A number is code x 2^(s - 127): an element of 4 bits (e2m1) or 8 bits (e4m3) and one scale byte s (e8m0, 255 = NaN)
// for each block of 32 along the contracted axis.  An operand of `rows` vectors of length k (times `groups`, for
// experts) is laid out once for the tensor cores:
//   codes   [group][row][kp] with kp = k rounded up to 128, contiguous along k (e2m1: two codes a byte, the even one
//           in the lower half); the codes from k to kp are zero, but for those behind NaN (a block with the NaN scale
//           ends with its 32 codes, a row of NaN from the norm with kp), which nothing reads.  One TMA box row is 128 bytes.
//   scales  [group][row tile of 128][k tile of 128][512]: the byte of row r and block b of a tile sits at
//           16 (r % 32) + 4 (r / 32) + b, which is what one tcgen05.cp 32x128b.warpx4 lays into TMEM as the scales of
//           128 rows; a k step of the product reads its scales as one contiguous copy per row tile.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>

#include "ozk_common.cuh"

namespace ozk_mx {

constexpr int BLOCK = 32;        // elements that share a scale
constexpr int TILE = 128;        // rows and elements of one scale tile
constexpr int TILE_BYTES = 512;  // scale bytes of one tile

__host__ __device__ constexpr int padded_k(int k) { return (k + TILE - 1) / TILE * TILE; }
__host__ __device__ constexpr int row_tiles(int rows) { return (rows + TILE - 1) / TILE; }
__host__ __device__ constexpr long long code_pitch(int fmt, int k) {
    return fmt == OZK_MX_E2M1 ? padded_k(k) / 2 : padded_k(k);
}
__host__ __device__ constexpr long long scale_group_bytes(int rows, int k) {
    return (long long)row_tiles(rows) * (padded_k(k) / TILE) * TILE_BYTES;
}
__device__ __forceinline__ int scale_slot(int row_in_tile, int block) {
    return (row_in_tile & 31) * 16 + (row_in_tile >> 5) * 4 + block;
}

// Scale byte of a block from the bit pattern of its largest magnitude (FP32): floor(log2 max) - emax + 127, which
// puts the largest number into [2^emax, 2^(emax + 1)) and saturates what lies above the format's largest number;
// `up`: one more where that would saturate.  Clamped at 0 (2^-127); 255 when a value is infinite or NaN.
template <int FMT>
__device__ __forceinline__ int block_scale(uint32_t max_bits, bool up) {
    constexpr int emax = FMT == OZK_MX_E2M1 ? 2 : 8;
    constexpr uint32_t top = FMT == OZK_MX_E2M1 ? 0x400000u : 0x600000u;   // mantissa of 6 = 1.5 x 4, of 448 = 1.75 x 256
    if (max_bits >= 0x7f800000u) return 255;
    const int s = (int)(max_bits >> 23) - emax + ((up && (max_bits & 0x7fffffu) > top) ? 1 : 0);
    return s < 0 ? 0 : s;
}

// 2^(127 - s), exact for every scale that block_scale gives except NaN (0 there: the codes are overwritten)
__device__ __forceinline__ float scale_inverse(int s) { return s == 255 ? 0.0f : __uint_as_float((uint32_t)(254 - s) << 23); }

// 2^(s - 127) for any scale byte (a subnormal for s = 0, NaN for 255)
__device__ __forceinline__ float scale_value(int s) {
    return __uint_as_float(s == 0 ? 0x00400000u : s == 255 ? 0x7fc00000u : (uint32_t)s << 23);
}

// Eight consecutive values, already multiplied by 2^(127 - s), to codes: 4 bytes (e2m1) or 8 (e4m3); to the nearest
// number of the format, ties to even, saturating.  A block without a scale (NaN or infinite values in it) gets the
// NaN code in e4m3 and the largest one in e2m1, which has no NaN: its scale says it.
template <int FMT>
__device__ __forceinline__ uint2 encode8(const float (&v)[8], bool bad) {
    uint2 out = make_uint2(0u, 0u);
    if (FMT == OZK_MX_E2M1) {
#pragma unroll
        for (int j = 0; j < 4; j++)
            out.x |= (uint32_t)__nv_cvt_float2_to_fp4x2(make_float2(v[2 * j], v[2 * j + 1]), __NV_E2M1, cudaRoundNearest)
                     << (8 * j);
        if (bad) out.x = 0x77777777u;
    } else {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++)
            w[j] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[2 * j], v[2 * j + 1]), __NV_SATFINITE, __NV_E4M3);
        out = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
        if (bad) out = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
    }
    return out;
}

// The eight element values that `encode8`'s codes stand for, exact in FP32
template <int FMT>
__device__ __forceinline__ void decode8(uint2 c, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        __half2_raw h;
        if (FMT == OZK_MX_E2M1) {
            h = __nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)(c.x >> (8 * j)), __NV_E2M1);
        } else {
            const uint32_t w = j < 2 ? c.x : c.y;
            h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * (j & 1))), __NV_E4M3);
        }
        const float2 f = __half22float2(__half2(h));
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
    }
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// the two 16-bit values of a 32-bit word (the tag pointer names the type), and back
__device__ __forceinline__ float2 unpack2(uint32_t w, const __half*) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ float2 unpack2(uint32_t w, const __nv_bfloat16*) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, const __half*) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, const __nv_bfloat16*) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Eight consecutive values as FP32.  `whole`: p is 16-byte aligned and all eight are inside; else the first `count`
// are read one by one (the others are 0).
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ p, bool whole, int count, float (&v)[8]) {
    if (whole) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 f = unpack2(w[j], (const T*)nullptr);
                v[2 * j] = f.x;
                v[2 * j + 1] = f.y;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = j < count ? to_f32(p[j]) : 0.0f;
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* __restrict__ p, bool whole, int count, const float (&v)[8]) {
    if (whole) {
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            const T* const type = nullptr;
            *reinterpret_cast<uint4*>(p) = make_uint4(pack2(v[0], v[1], type), pack2(v[2], v[3], type),
                                                      pack2(v[4], v[5], type), pack2(v[6], v[7], type));
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j < count) p[j] = from_f32<T>(v[j]);
    }
}

// ---- rows that start anywhere ----
// The lanes of a row read the aligned 16 bytes ("granules") that cover it, each its own, get the next one from their
// neighbour and shift the two into place.  Granules from a row's end on are not read; of the others the matrix's first and
// last may reach out of it, and are read value by value: bytes outside [begin, end) never are.
__device__ __forceinline__ uint4 load_granule(uintptr_t at, uintptr_t row_end, uintptr_t begin, uintptr_t end) {
    if (at >= row_end) return make_uint4(0u, 0u, 0u, 0u);
    if (at >= begin && at + 16 <= end) return __ldg(reinterpret_cast<const uint4*>(at));
    uint16_t e[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const uintptr_t p = at + 2 * j;
        e[j] = p >= begin && p < end ? __ldg(reinterpret_cast<const unsigned short*>(p)) : (uint16_t)0;
    }
    return make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16,
                      e[6] | (uint32_t)e[7] << 16);
}
// the first `count` of eight 16-bit values, zeros behind
__device__ __forceinline__ uint4 keep8(uint4 w, int count) {
    if (count >= 8) return w;
    uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; j++) u[j] = count >= 2 * j + 2 ? u[j] : count == 2 * j + 1 ? u[j] & 0xffffu : 0u;
    return make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ uint4 next_lane(uint4 g) {
    return make_uint4(__shfl_down_sync(0xffffffffu, g.x, 1), __shfl_down_sync(0xffffffffu, g.y, 1),
                      __shfl_down_sync(0xffffffffu, g.z, 1), __shfl_down_sync(0xffffffffu, g.w, 1));
}
// the 16 bytes from byte `sh` (0, 2 .. 14) of the 32 that g and n hold
__device__ __forceinline__ uint4 shift_granules(uint4 g, uint4 n, uint32_t sh) {
    uint32_t w[8] = {g.x, g.y, g.z, g.w, n.x, n.y, n.z, n.w};
    if (sh & 8u) {
#pragma unroll
        for (int j = 0; j < 6; j++) w[j] = w[j + 2];
    }
    if (sh & 4u) {
#pragma unroll
        for (int j = 0; j < 5; j++) w[j] = w[j + 1];
    }
    if (sh & 2u) {
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = __funnelshift_r(w[j], w[j + 1], 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// the larger magnitude, NaN if either is
__device__ __forceinline__ float max_magnitude(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(fabsf(a)), "f"(fabsf(b)));
    return m;
}

// bits of the largest magnitude of eight values (at least those of infinity if one is infinite or NaN)
__device__ __forceinline__ uint32_t max_bits8(const float (&v)[8]) {
    const float a = max_magnitude(max_magnitude(v[0], v[1]), max_magnitude(v[2], v[3]));
    const float b = max_magnitude(max_magnitude(v[4], v[5]), max_magnitude(v[6], v[7]));
    return __float_as_uint(max_magnitude(a, b));
}

// largest of the four lanes that hold one block (lanes 4 i .. 4 i + 3)
__device__ __forceinline__ uint32_t quad_max(uint32_t m) {
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    return max(m, __shfl_xor_sync(0xffffffffu, m, 2));
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline bool dtype_ok(int dtype) { return dtype == OZK_F32 || dtype == OZK_F16 || dtype == OZK_BF16; }
// p points at values of that (valid) type: a null pointer does too
inline bool on_elements(const void* p, int dtype) { return (reinterpret_cast<uintptr_t>(p) & (dtype == OZK_F32 ? 3 : 1)) == 0; }
inline bool fmt_ok(int fmt) { return fmt == OZK_MX_E2M1 || fmt == OZK_MX_E4M3; }

}  // namespace ozk_mx
