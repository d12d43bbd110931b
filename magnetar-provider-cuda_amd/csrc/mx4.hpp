// The 4-bit store: f32 rows [capacity, kv_heads * d] held as codes of four
// bits (E2M1: sign, two exponent bits, one fraction bit; the values 0, 0.5, 1,
// 1.5, 2, 3, 4 and 6), each block of 32 values of a head under one E8M0 scale
// byte s, 2^(s - 127) (255: not a number). 17/32 of a byte a value.
//
// Both are formats that gfx950 converts in hardware (two codes and a scale to
// two bf16 or f32 in one instruction, and back), and every held value is a
// bf16 exactly: its two fraction bits and exponents from -121 to 127.
//
// Layout, for NB = ceil(d / 32) blocks a head and G = ceil(capacity / 4) groups
// of four rows:
//
//   codes  [kv_heads][G][16 lanes n][4 rows][NB bytes p]
//   scales [kv_heads][G][NB blocks p][4 rows], one byte each
//
// rounded up to 256 bytes. Byte (n, row, p) holds the codes of the head's
// values 32 p + n (low four bits) and 32 p + 16 + n (high): the two share a
// scale, which one conversion takes. A unit (head, group, n) is NB dwords with
// all four rows of its 2 NB columns, and for a token's few rows both products of
// attention are fed from whole units, with no pass through LDS
// (attention_mx4.hip). A head's rows are contiguous, so a chunk of keys is one
// stretch of memory.
#pragma once

#include "common.hpp"

namespace mhip {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr uint64_t kMx4MaxDimension = 256;
constexpr uint32_t kMx4NaN = 255;

inline uint64_t mx4_blocks(uint64_t d) { return ceil_div(d, 32); }
inline uint64_t mx4_groups(uint64_t capacity) { return ceil_div(capacity, 4); }
// Bytes of the codes, after which the scales begin.
inline uint64_t mx4_code_bytes(uint64_t capacity, uint64_t heads, uint64_t d) {
    return heads * mx4_groups(capacity) * 64 * mx4_blocks(d);
}
// Bytes in use, and as allocated: consecutive stores stay 256-byte aligned.
inline uint64_t mx4_used_bytes(uint64_t capacity, uint64_t heads, uint64_t d) {
    return heads * mx4_groups(capacity) * 68 * mx4_blocks(d);
}
inline uint64_t mx4_bytes(uint64_t capacity, uint64_t heads, uint64_t d) {
    return (mx4_used_bytes(capacity, heads, d) + 255) / 256 * 256;
}

// Checks a store's shape; `what` names the call.
mhip_status mx4_check(const mhip_mx4_store* s, const char* what);

// The conversions' scale operand from byte `row` (a constant) of a scale
// dword: they read its exponent field alone, so the other bits may hold the
// neighbours.
__device__ __forceinline__ float mx4_scale(uint32_t dword, int row) {
    return __uint_as_float(row == 3 ? dword >> 1 : dword << (23 - 8 * row));
}

// The two values of byte `sel` (a constant) of `codes`, low half first.
__device__ __forceinline__ bf16x2 mx4_bf16(uint32_t codes, float scale, int sel) {
    switch (sel) {
        case 0: return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
        case 1: return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
        case 2: return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
        default: return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
    }
}
__device__ __forceinline__ f32x2 mx4_f32(uint32_t codes, float scale, int sel) {
    switch (sel) {
        case 0: return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 0);
        case 1: return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 1);
        case 2: return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 2);
        default: return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 3);
    }
}

// NB dwords of a unit (codes) or of a group's scales: 4-byte aligned, which
// is all that a wide global load asks for.
template <int NB>
struct Mx4Unit {
    uint32_t w[NB];
};
template <int NB>
__device__ __forceinline__ Mx4Unit<NB> mx4_load(const uint32_t* p) {
    Mx4Unit<NB> u;
    __builtin_memcpy(&u, __builtin_assume_aligned(p, NB % 4 == 0 ? 16 : NB % 2 == 0 ? 8 : 4), sizeof(u));
    return u;
}

}  // namespace mhip
