// What the products of 4-bit matrices share: how rows are given, and a matrix's numbers as operands.
#pragma once

#include "common.h"
#include "epilogue.h"
#include "mx.h"

namespace liyab {

typedef __attribute__((ext_vector_type(8))) __bf16 mx_bf16x8;

enum : int { kRowsBF16 = 0, kRowsF32 = 1, kRowsMx = 2 };

struct MxRowsIn {
    const void* a;          // [M, lda], bfloat16, float32 or codes
    int64_t lda;            // elements
    const uint8_t* scales;  // [M, lds] of rows in 8 bits
    int64_t lds;
};

// What a load behind a row's end reads instead: zeros, so that the zeros of the matrix there meet numbers. (One value, aligned as loads of 16 bytes take it.)
typedef __attribute__((ext_vector_type(4))) uint32_t mx_u32x4;
static __device__ __constant__ const mx_u32x4 kMxZeros = {0, 0, 0, 0};
__device__ __forceinline__ const mx_u32x4* mx_zeros() { return &kMxZeros; }

// Eight numbers of a block's row as bfloat16, scale and all: exact.
__device__ __forceinline__ mx_bf16x8 mx_eight_of(uint32_t word, float power) {
    const mx_bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, power, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, power, 1),
                    c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, power, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, power, 3);
    return mx_bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Eight numbers of a row in 8 bits as bfloat16, scale and all: three bits of mantissa and a power of two, exact (where bfloat16 has their magnitude: from scales of
// 2^-124 on all of them, and up to 2^127).
__device__ __forceinline__ mx_bf16x8 mx_eight_of_rows(uint32_t lo, uint32_t hi, float power) {
    const mx_bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, power, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, power, true),
                    c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, power, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, power, true);
    return mx_bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// mx_tiles.hip: products of many rows in bfloat16 or 8 bits, in tiles of 64 x 128, 128 x 128, 128 x 256 or 256 x 256.
enum : int { kMxTile128 = 1, kMxTile256 = 2, kMxTile64 = 3, kMxTileWide = 4 };
int launch_mx_tiles(int kind, int tile, const MxRowsIn& in, const uint8_t* blocks, int M, int N, int K, const EpiParams& epi, hipStream_t stream);

}  // namespace liyab
