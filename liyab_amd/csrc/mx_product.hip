// out[M, N] = rows[M, K] . matrix[N, K]^T with the matrix in 4 bits (mx.h) and rows in bfloat16, float32 or 8 bits; the waves of a
// workgroup share K.
//
// A wave reads blocks of 16 matrix rows and 128 k as they lie in memory, 17 bytes a lane, and rows straight from the caches: no
// LDS stands between memory and the matrix instructions. What a lane holds of a block are 32 neighbouring k of one matrix row, and it takes
// the same 32 k of its row of activations (the order in which an instruction goes through k is the same for both operands):
//   bfloat16  two numbers a conversion, the group's scale with them, exact; four 16x16x32 instructions
//   float32   the same in 32 bits; 32 16x16x4 instructions: chains of fused multiply-adds in 32 bits
//   8 bits    the rows' numbers become bfloat16 too (three bits of mantissa and a power of two: exact), then as above. The scaled instruction
//             takes them as they are, but adds eight neighbouring products without the bits that lie 14 places below the largest: sums
//             of 32 bits, as here, cost nothing where memory sets the pace
// Chunk c of K goes to wave c % waves; the waves' sums meet in LDS in the waves' order.
#include "common.h"
#include "epilogue.h"
#include "launchers.h"
#include "mx.h"
#include "mx_product.h"

namespace liyab {

typedef __attribute__((ext_vector_type(4))) float mx_f32x4;

// A chunk of one row as the matrix instructions take it.
template <int ROWS>
struct MxRowPart;
template <>
struct MxRowPart<kRowsBF16> {
    uint4 piece[4];
    __device__ __forceinline__ mx_bf16x8 eight(int j) const { return __builtin_bit_cast(mx_bf16x8, piece[j]); }
};
template <>
struct MxRowPart<kRowsF32> {
    uint4 piece[8];
};
template <>
struct MxRowPart<kRowsMx> {
    uint4 piece[2];
    uint32_t scale;
    __device__ __forceinline__ mx_bf16x8 eight(int j) const {
        const uint4 p = piece[j / 2];
        const uint32_t lo = j % 2 == 0 ? p.x : p.z, hi = j % 2 == 0 ? p.y : p.w;
        const float power = mx_power(scale);
        const mx_bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, power, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, power, true),
                        c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, power, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, power, true);
        return mx_bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
};

// TAIL: K is no multiple of 128 (it is one of the 8 or 4 elements of a piece).
template <int ROWS, bool TAIL>
__device__ __forceinline__ void load_row(MxRowPart<ROWS>& part, const uint8_t* row, const uint8_t* scales, int c, int g, int K) {
    if constexpr (ROWS == kRowsMx) {
        const uint8_t* p = row + c * kMxChunk + kMxGroup * g;
        part.piece[0] = *reinterpret_cast<const uint4*>(p);
        part.piece[1] = *reinterpret_cast<const uint4*>(p + 16);
        part.scale = scales[4 * c + g];
    } else {
        constexpr int SIZE = ROWS == kRowsBF16 ? 2 : 4, PER = 16 / SIZE;
        const int k = c * kMxChunk + kMxGroup * g;
#pragma unroll
        for (int j = 0; j < kMxGroup / PER; ++j) {
            const uint8_t* p = row + static_cast<int64_t>(k + j * PER) * SIZE;
            if (TAIL && k + j * PER >= K) p = reinterpret_cast<const uint8_t*>(mx_zeros());
            part.piece[j] = *reinterpret_cast<const uint4*>(p);
        }
    }
}

// acc[i] += matrix rows 4 g + i of the block times the lane's row.
template <int ROWS, int MT>
__device__ __forceinline__ void multiply_block(mx_f32x4 (&acc)[MT], const uint4& codes, uint32_t scale, const MxRowPart<ROWS> (&rows)[MT]) {
    const uint32_t word[4] = {codes.x, codes.y, codes.z, codes.w};
    if constexpr (ROWS != kRowsF32) {
        const float power = mx_power(scale);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const mx_bf16x8 w = mx_eight_of(word[j], power);
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, rows[t].eight(j), acc[t], 0, 0, 0);
        }
    } else {
        const float power = mx_power(scale);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const mx_f32x2 w[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[j], power, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[j], power, 1),
                                   __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[j], power, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[j], power, 3)};
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    const uint4 x = rows[t].piece[2 * j + i / 4];
                    const float xv = __uint_as_float(i % 4 == 0 ? x.x : i % 4 == 1 ? x.y : i % 4 == 2 ? x.z : x.w);
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[i / 2][i % 2], xv, acc[t], 0, 0, 0);
                }
        }
    }
}

// MT tiles of 16 rows and NS strips of the matrix a workgroup of blockDim.x / 64 waves.
template <int ROWS, int MT, int NS, int UNROLL, bool TAIL, int MAXW>
__global__ void __launch_bounds__(64 * MAXW)
mx_product_kernel(MxRowsIn in, const uint8_t* __restrict__ blocks, int M, int N, int K, int strips, EpiParams epi) {
    extern __shared__ __attribute__((aligned(16))) float red[];
    constexpr int LDN = 16 * NS + 4;  // floats a row of the sums in LDS
    constexpr int SIZE = ROWS == kRowsBF16 ? 2 : ROWS == kRowsF32 ? 4 : 1;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
    const int g = lane / 16, r = lane % 16;
    const int strip0 = blockIdx.x * NS, m0 = blockIdx.y * 16 * MT;
    const int chunks = mx_chunks(K);

    const uint8_t* row[MT];
    const uint8_t* row_scales[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int64_t m = min(m0 + 16 * t + r, M - 1);
        row[t] = static_cast<const uint8_t*>(in.a) + m * in.lda * SIZE;
        row_scales[t] = ROWS == kRowsMx ? in.scales + m * in.lds : nullptr;
    }
    const uint8_t* block[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) block[s] = blocks + static_cast<int64_t>(min(strip0 + s, strips - 1)) * chunks * kMxBlockBytes;

    mx_f32x4 acc[NS][MT];
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[s][t] = mx_f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    for (int c0 = wave; c0 < chunks; c0 += waves * UNROLL) {
        uint4 codes[UNROLL][NS];
        uint32_t scale[UNROLL][NS];
        MxRowPart<ROWS> part[UNROLL][MT];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int c = min(c0 + u * waves, chunks - 1);  // (a chunk past the end is read and not multiplied)
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                const uint8_t* b = block[s] + static_cast<int64_t>(c) * kMxBlockBytes;
                codes[u][s] = *reinterpret_cast<const uint4*>(b + 16 * lane);
                scale[u][s] = b[1024 + lane];
            }
#pragma unroll
            for (int t = 0; t < MT; ++t) load_row<ROWS, TAIL>(part[u][t], row[t], row_scales[t], c, g, K);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (c0 + u * waves < chunks) {
#pragma unroll
                for (int s = 0; s < NS; ++s) multiply_block<ROWS, MT>(acc[s], codes[u][s], scale[u][s], part[u]);
            }
    }

    // the waves' sums, added in the waves' order; a wave's tile in LDS: row m, then the strips' columns
    constexpr int TILE = MT * 16 * LDN;
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int t = 0; t < MT; ++t) *reinterpret_cast<mx_f32x4*>(red + wave * TILE + (16 * t + r) * LDN + 16 * s + 4 * g) = acc[s][t];
    __syncthreads();
    for (int i = threadIdx.x; i < MT * 16 * 16 * NS; i += blockDim.x) {
        const int ml = i / (16 * NS), nl = i % (16 * NS);
        const int m = m0 + ml, n = strip0 * 16 + nl;
        if (m >= M || n >= N) continue;
        float v = 0.0f;
        for (int w = 0; w < waves; ++w) v += red[w * TILE + ml * LDN + nl];
        if (epi.out_dtype == kBF16) epilogue_store<bf16_t, -1, ROWS == kRowsF32>(epi, m, n, v);
        else epilogue_store<float, -1, ROWS == kRowsF32>(epi, m, n, v);
    }
}

template <int ROWS, int MT, int NS, int UNROLL, int MAXW>
static int launch_product(const MxRowsIn& in, const uint8_t* blocks, int M, int N, int K, const EpiParams& epi, hipStream_t stream) {
    const int strips = mx_strips(N), chunks = mx_chunks(K);
    const int waves = chunks < MAXW ? chunks : MAXW;
    const int64_t tiles = (M + 16 * MT - 1) / (16 * MT);
    LIYAB_REQUIRE(tiles <= 65535, "mx_product: %d rows are too many", M);
    const dim3 grid(static_cast<unsigned>((strips + NS - 1) / NS), static_cast<unsigned>(tiles));
    const size_t lds = sizeof(float) * waves * MT * 16 * (16 * NS + 4);
    auto* kernel = ROWS != kRowsMx && K % kMxChunk != 0 ? &mx_product_kernel<ROWS, MT, NS, UNROLL, ROWS != kRowsMx, MAXW>
                                                        : &mx_product_kernel<ROWS, MT, NS, UNROLL, false, MAXW>;
    kernel<<<grid, 64 * waves, lds, stream>>>(in, blocks, M, N, K, strips, epi);
    return check_launch("mx_product");
}

template <int ROWS>
static int product_of_rows(int tile, const MxRowsIn& in, const uint8_t* blocks, int M, int N, int K, const EpiParams& epi, hipStream_t stream) {
    if (tile >= 0 && (M > 64 || tile > 0) && ROWS != kRowsF32) return launch_mx_tiles(ROWS, tile, in, blocks, M, N, K, epi, stream);
    if (M <= 16) return launch_product<ROWS, 1, 1, 2, 8>(in, blocks, M, N, K, epi, stream);
    if (M <= 32) return launch_product<ROWS, 2, 1, 1, 8>(in, blocks, M, N, K, epi, stream);
    return launch_product<ROWS, 4, 1, 1, 8>(in, blocks, M, N, K, epi, stream);
}

}  // namespace liyab

using namespace liyab;

// a: rows [M, lda] of `rows` 0: bfloat16, 1: float32, 2: e4m3 codes (padded with zeros to whole chunks) with their scales [M, lds].
// tile: 0 chooses the kernel from the sizes, -1 takes this file's whatever they are (one order of every sum, so that a row's bits follow K alone), a positive
// number a tile of mx_tiles.hip.
extern "C" int liyab_mx_product(const void* a, int64_t lda, const void* a_scales, int64_t lds, int rows, const void* blocks, int M, int N, int K, int tile,
                                const EpiParams* epi, hipStream_t stream) {
    LIYAB_REQUIRE(a && blocks && epi, "mx_product: null pointer");
    LIYAB_REQUIRE(M >= 0 && N > 0 && K > 0, "mx_product: bad sizes");
    if (M == 0) return 0;
    if (const int rc = check_epilogue(*epi, M, N)) return rc;
    LIYAB_REQUIRE(epi->out_dtype == kF32 || epi->out_dtype == kBF16, "mx_product: unknown output dtype %d", epi->out_dtype);
    LIYAB_REQUIRE(reinterpret_cast<uintptr_t>(a) % 16 == 0 && reinterpret_cast<uintptr_t>(blocks) % 16 == 0, "mx_product: operands start on 16-byte boundaries");
    const MxRowsIn in{a, lda, static_cast<const uint8_t*>(a_scales), lds};
    const uint8_t* const b = static_cast<const uint8_t*>(blocks);
    if (rows == kRowsMx) {
        LIYAB_REQUIRE(a_scales && lda >= static_cast<int64_t>(mx_chunks(K)) * kMxChunk && lda % 16 == 0 && lds >= mx_chunks(K) * 4, "mx_product: rows in 8 bits are padded to %d codes",
                      mx_chunks(K) * kMxChunk);
        return product_of_rows<kRowsMx>(tile, in, b, M, N, K, *epi, stream);
    }
    const int per = rows == kRowsBF16 ? 8 : 4;
    LIYAB_REQUIRE(rows == kRowsBF16 || rows == kRowsF32, "mx_product: unknown kind of rows %d", rows);
    LIYAB_REQUIRE(K % per == 0 && lda % per == 0 && lda >= K, "mx_product: rows of whole pieces of 16 bytes are taken (K = %d, row stride %lld)", K, static_cast<long long>(lda));
    return rows == kRowsBF16 ? product_of_rows<kRowsBF16>(tile, in, b, M, N, K, *epi, stream) : product_of_rows<kRowsF32>(tile, in, b, M, N, K, *epi, stream);
}
