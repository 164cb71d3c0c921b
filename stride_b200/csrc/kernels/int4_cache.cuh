// Rows of a cache that holds keys and values in 4 bits.
//
// A row (one head of one token) is cut into groups of 32 neighbouring entries, the last one possibly shorter. A group has a scale s and
// a centre c, both bfloat16, and a number n in 0 .. 15 for each entry, which stands for c + s (n - 8):
//     s = bf16((max - min) / 15)      c = bf16(min + 8 s)      n = clamp(rint((x - c) / s) + 8, 0, 15)      (s = 0: n = 8)
// so an entry is off by half a step, and at the ends of the range by what c is rounded by, up to 2^-8 |c|, and at the upper one by 15 times what s
// is, up to 2^-8 s each: a group whose entries lie close together far from zero (100 to 100.1: c = 100, s = 0.0067) keeps few of its 4 bits.
// 5 bits an entry.
// A row of G groups is 16 G bytes of numbers, then (s, c) of each group, 4 bytes a group: 20 G bytes, whatever the head size.
// The numbers lie as the lanes of a matrix instruction want them, without a shuffle:
//   keys    entry 8 a + i of group g: 32-bit word a G + g, bits 4 i      (a lane that takes part a = lane % 4 of every key finds it side by side)
//   values  entry 4 a + i of group g: 16-bit word a G + g, bits 4 i      (a lane that takes part a = lane / 4 of every value, likewise)
// A number that stands for nothing (behind a head's last entry) is 8.
// A key or value that is no number or not below 2^64 makes its token no number for that key head: the key row gets s = c = NaN and the value
// row zeros, so whoever sees the token gets NaN and whoever does not is left alone, whatever the mask multiplies. (Below 2^64 a weight
// can be scaled against a row's scales and centres without leaving the 32-bit range.)
#pragma once

#include <cstring>

#include "common.cuh"

namespace stride {

// A launcher's arguments as one record that the caller packs.
template <typename R>
inline R read_record(const void* record) {
    R r;
    std::memcpy(&r, record, sizeof(R));
    return r;
}

namespace four {

constexpr int kGroup = 32;
constexpr int kMaxHeadDim = 256;
constexpr int kMaxGroups = kMaxHeadDim / kGroup;
constexpr float kMaxEntry = 1.8446744e19f;      // 2^64

__host__ __device__ __forceinline__ int groups_of(int hd) { return (hd + kGroup - 1) / kGroup; }
__host__ __device__ __forceinline__ int row_bytes(int hd) { return 20 * groups_of(hd); }

// The codes that a kernel leaves in the status word.
constexpr int kCodeNoPage = 33;         // a key's page is not one of the cache's
constexpr int kCodeNoSlot = 34;         // a token's slot lies behind the cache's last page
constexpr int kCodeTooManyKeys = 36;    // the requests hold more keys than the launch was told
constexpr int kCodeNoPosition = 35;     // a token's position lies behind the rotation's tables

__device__ __forceinline__ void complain(int* status, int code) {
    if (status != nullptr) atomicCAS(status, 0, code);
}

__device__ __forceinline__ float bf16_low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack_params(float s, float c) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(s, c);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// s (rounded to bfloat16) and c (likewise) of a group whose least and largest entries are lo and hi. The smallest scale that is kept
// is the smallest normal number: below it 1 / s would not be finite.
__device__ __forceinline__ void group_params(float lo, float hi, float& s, float& c) {
    s = __bfloat162float(__float2bfloat16_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f)));
    if (s < 1.17549435e-38f) s = 0.f;       // (a NaN passes on)
    c = __bfloat162float(__float2bfloat16_rn(__fadd_rn(lo, __fmul_rn(8.f, s))));
}

__device__ __forceinline__ uint32_t number_of(float x, float c, float inverse) {
    return static_cast<uint32_t>(fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(x, c), inverse)) + 8.f, 0.f), 15.f));
}

__device__ __forceinline__ float value_of(uint32_t n, float s, float c) {
    return __fadd_rn(c, __fmul_rn(s, static_cast<float>(static_cast<int>(n) - 8)));
}

}  // namespace four
}  // namespace stride
