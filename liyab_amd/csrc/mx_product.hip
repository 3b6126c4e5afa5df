// out[M, N] = rows[M, K] . matrix[N, K]^T with the matrix in 4 bits (mx.h) and rows in bfloat16, float32 or 8 bits, for few rows: the waves of a
// workgroup share K.
//
// A wave reads blocks of 16 matrix rows and 128 k as they lie in memory, 17 bytes a lane, into registers. What a lane holds of a block are 32
// neighbouring k of one matrix row, and it takes the same 32 k of its row of activations (the order in which an instruction goes
// through k is the same for both operands). Rows come through a stretch of LDS that is the wave's own: a direct load (16 bytes a lane) brings whole
// stretches of a few rows, where lanes that read their own rows from the caches touch a line each (64 rows, 16,384 -> 4,096: 74 us). UNROLL chunks
// of rows and matrix are in flight while the UNROLL before them, by then in registers, are multiplied; no wave waits for another until the end.
//   bfloat16  two numbers a conversion, the group's scale with them, exact; four 16x16x32 instructions
//   float32   the same in 32 bits; 32 16x16x4 instructions: chains of fused multiply-adds in 32 bits
//   8 bits    the rows' numbers become bfloat16 too (three bits of mantissa and a power of two: exact), then as above
// Chunk c of K goes to wave c % waves; the waves' sums meet in LDS in the waves' order.
#include "common.h"
#include "epilogue.h"
#include "launchers.h"
#include "mx.h"
#include "mx_product.h"

#include <atomic>

namespace liyab {

typedef __attribute__((ext_vector_type(4))) float mx_f32x4;
typedef __attribute__((address_space(3))) void* mx_lds_ptr;

// A chunk of a row: its bytes, 16-byte pieces, and how many rows one load of 64 lanes brings.
template <int ROWS>
struct MxRowShape {
    static constexpr int BYTES = ROWS == kRowsMx ? 128 : ROWS == kRowsBF16 ? 256 : 512;
    static constexpr int PIECES = BYTES / 16, ROWS_A_LOAD = kWave / PIECES, PIECES_A_GROUP = PIECES / 4;
    // Where a row's pieces sit in LDS (piece ^ place), so that 16 lanes' reads of 16 rows at one piece fall into different banks.
    static __device__ __forceinline__ int place(int row) { return ROWS == kRowsMx ? (row >> 1) & 7 : row & 15; }
};

// What a lane holds of a chunk of its row: the 32 k of its group.
template <int ROWS>
struct MxRowPart {
    uint4 piece[MxRowShape<ROWS>::PIECES_A_GROUP];
    uint32_t scale;  // of rows in 8 bits

    // Eight k, 8 j and on, as bfloat16.
    __device__ __forceinline__ mx_bf16x8 eight(int j) const {
        if constexpr (ROWS == kRowsBF16) {
            return __builtin_bit_cast(mx_bf16x8, piece[j]);
        } else {
            const uint4 p = piece[j / 2];
            const uint32_t lo = j % 2 == 0 ? p.x : p.z, hi = j % 2 == 0 ? p.y : p.w;
            return mx_eight_of_rows(lo, hi, mx_power(scale));
        }
    }
};

// acc[s][t] += matrix rows of strip s (4 g + i in element i) times the lane's row of tile t.
template <int ROWS, int MT, int NS>
__device__ __forceinline__ void multiply_chunk(mx_f32x4 (&acc)[NS][MT], const uint4 (&codes)[NS], const uint32_t (&scale)[NS], const MxRowPart<ROWS> (&rows)[MT]) {
    if constexpr (ROWS != kRowsF32) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            mx_bf16x8 x[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) x[t] = rows[t].eight(j);
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                const mx_bf16x8 w = mx_eight_of(j == 0 ? codes[s].x : j == 1 ? codes[s].y : j == 2 ? codes[s].z : codes[s].w, mx_power(scale[s]));
#pragma unroll
                for (int t = 0; t < MT; ++t) acc[s][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x[t], acc[s][t], 0, 0, 0);
            }
        }
    } else {
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t word = j == 0 ? codes[s].x : j == 1 ? codes[s].y : j == 2 ? codes[s].z : codes[s].w;
                const float power = mx_power(scale[s]);
                const mx_f32x2 w[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, power, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, power, 1),
                                       __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, power, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, power, 3)};
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        const uint4 x = rows[t].piece[2 * j + i / 4];
                        const float xv = __uint_as_float(i % 4 == 0 ? x.x : i % 4 == 1 ? x.y : i % 4 == 2 ? x.z : x.w);
                        acc[s][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[i / 2][i % 2], xv, acc[s][t], 0, 0, 0);
                    }
            }
    }
}

// MT tiles of 16 rows and NS strips of the matrix a workgroup of blockDim.x / 64 waves; `row_loads`: loads that bring a chunk of its rows.
template <int ROWS, int MT, int NS, int UNROLL, int MAXW>
__global__ void __launch_bounds__(64 * MAXW)
mx_product_kernel(MxRowsIn in, const uint8_t* __restrict__ blocks, int M, int N, int K, int strips, int row_loads, EpiParams epi) {
    using Shape = MxRowShape<ROWS>;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    constexpr int SIZE = ROWS == kRowsBF16 ? 2 : ROWS == kRowsF32 ? 4 : 1;
    constexpr int MAX_LOADS = MT * 16 / Shape::ROWS_A_LOAD;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), waves = blockDim.x / kWave;
    const int g = lane / 16, r = lane % 16;
    const int strip0 = blockIdx.x * NS, m0 = blockIdx.y * 16 * MT;
    const int chunks = mx_chunks(K);

    // this wave's stretch of LDS: UNROLL chunks of up to 16 MT rows; and this lane's part in a load: a row and the position of a piece in it
    uint8_t* const own = lds + wave * (UNROLL * row_loads * 1024);
    const int64_t stride = in.lda * SIZE;
    const uint8_t* row[MAX_LOADS];
    int piece[MAX_LOADS];
#pragma unroll
    for (int i = 0; i < MAX_LOADS; ++i) {
        const int m = i * Shape::ROWS_A_LOAD + lane / Shape::PIECES;
        row[i] = static_cast<const uint8_t*>(in.a) + min(m0 + m, M - 1) * stride;
        piece[i] = ((lane % Shape::PIECES) ^ Shape::place(m)) * 16;
    }
    const int64_t row_bytes = ROWS == kRowsMx ? static_cast<int64_t>(chunks) * kMxChunk : static_cast<int64_t>(K) * SIZE;
    const uint8_t* row_scales[ROWS == kRowsMx ? MT : 1];
    if constexpr (ROWS == kRowsMx) {
#pragma unroll
        for (int t = 0; t < MT; ++t) row_scales[t] = in.scales + min(m0 + 16 * t + r, M - 1) * in.lds + g;
    }
    const uint8_t* block[NS];  // (the same in every lane)
#pragma unroll
    for (int s = 0; s < NS; ++s) block[s] = blocks + static_cast<int64_t>(min(strip0 + s, strips - 1)) * chunks * kMxBlockBytes;

    uint4 codes[UNROLL][NS];
    uint32_t scale[UNROLL][NS];
    uint32_t next_scale[UNROLL][MT];
    auto issue = [&](int c0) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int c = min(c0 + u * waves, chunks - 1);  // (a chunk past the end is read and not multiplied)
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                const uint8_t* const b = block[s] + static_cast<int64_t>(c) * kMxBlockBytes;
                codes[u][s] = *reinterpret_cast<const uint4*>(b + static_cast<uint32_t>(16 * lane));
                scale[u][s] = b[1024 + static_cast<uint32_t>(lane)];
            }
            const int64_t at = static_cast<int64_t>(c) * Shape::BYTES;
#pragma unroll
            for (int i = 0; i < MAX_LOADS; ++i)
                if (i < row_loads) {
                    const uint8_t* src = row[i] + (at + piece[i]);
                    if (ROWS != kRowsMx && at + piece[i] >= row_bytes) src = reinterpret_cast<const uint8_t*>(mx_zeros());
                    __builtin_amdgcn_global_load_lds(src, (mx_lds_ptr)(own + (u * row_loads + i) * 1024), 16, 0, 0);
                }
            if constexpr (ROWS == kRowsMx) {
#pragma unroll
                for (int t = 0; t < MT; ++t) next_scale[u][t] = row_scales[t][4 * c];
            }
        }
    };

    mx_f32x4 acc[NS][MT];
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[s][t] = mx_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // (rows past the loaded ones: another row's numbers, whose results are not stored)
    int local[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) local[t] = min(16 * t + r, row_loads * Shape::ROWS_A_LOAD - 1);

    if (wave < chunks) issue(wave);
    for (int c0 = wave; c0 < chunks; c0 += waves * UNROLL) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        uint4 now_codes[UNROLL][NS];
        uint32_t now_scale[UNROLL][NS];
        MxRowPart<ROWS> part[UNROLL][MT];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                now_codes[u][s] = codes[u][s];
                now_scale[u][s] = scale[u][s];
            }
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const uint8_t* const from = own + u * row_loads * 1024 + local[t] * Shape::BYTES;
#pragma unroll
                for (int p = 0; p < Shape::PIECES_A_GROUP; ++p)
                    part[u][t].piece[p] = *reinterpret_cast<const uint4*>(from + ((Shape::PIECES_A_GROUP * g + p) ^ Shape::place(local[t])) * 16);
                if constexpr (ROWS == kRowsMx) part[u][t].scale = next_scale[u][t];
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stretch has been read
        if (c0 + waves * UNROLL < chunks) issue(c0 + waves * UNROLL);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (c0 + u * waves < chunks) multiply_chunk<ROWS, MT, NS>(acc, now_codes[u], now_scale[u], part[u]);
    }

    // the waves' sums, added in the waves' order; a wave's tile in LDS: row m, then the strips' columns
    constexpr int LDN = 16 * NS + 4, TILE = MT * 16 * LDN;
    float* const red = reinterpret_cast<float*>(lds);
    __syncthreads();
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
    const int64_t tiles = (static_cast<int64_t>(M) + 16 * MT - 1) / (16 * MT);
    LIYAB_REQUIRE(tiles <= 65535, "mx_product: %d rows are too many", M);
    const dim3 grid(static_cast<unsigned>((strips + NS - 1) / NS), static_cast<unsigned>(tiles));
    constexpr int PER = MxRowShape<ROWS>::ROWS_A_LOAD;
    const int row_loads = ((M < 16 * MT ? M : 16 * MT) + PER - 1) / PER;
    const size_t ring = static_cast<size_t>(waves) * UNROLL * row_loads * 1024, sums = sizeof(float) * waves * MT * 16 * (16 * NS + 4);
    constexpr size_t MOST = 160 * 1024;
    static_assert(static_cast<size_t>(MAXW) * UNROLL * (MT * 16 / PER) * 1024 <= MOST && sizeof(float) * MAXW * MT * 16 * (16 * NS + 4) <= MOST, "LDS");
    auto* kernel = &mx_product_kernel<ROWS, MT, NS, UNROLL, MAXW>;
    static std::atomic<bool> ready{false};  // once a kernel
    if (!ready.load(std::memory_order_relaxed)) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, MOST);
        if (e != hipSuccess) return fail(2, "mx_product: %s", hipGetErrorString(e));
        ready.store(true, std::memory_order_relaxed);
    }
    kernel<<<grid, 64 * waves, ring > sums ? ring : sums, stream>>>(in, blocks, M, N, K, strips, row_loads, epi);
    return check_launch("mx_product");
}

// The workgroups' shapes: tiles of 16 rows x strips of 16 columns, and the tiles of mx_tiles.hip.
enum : int { kShape1x1 = 11, kShape1x2 = 12, kShape2x1 = 21, kShape2x2 = 22, kShape2x4 = 24, kShape4x1 = 41, kShape4x2 = 42, kShape4x4 = 44 };

// The shape that takes the least time: `fixed` and another `round` for each round of 256 workgroups, in us at 4,096 k (bfloat16 / 8-bit rows; measured over
// matrices that are not in the caches, 24 to 2,048 rows of 768 to 16,384 columns; K changes them all much alike). The shapes of this file fill a compute unit
// each; the smaller tiles leave room for others, so their rounds run into each other. What it chooses between, us: 512 rows 4,096 x 4,096 4x4 / 64 x 128
// / 128 x 128 bfloat16 32 / 29 / 38, 8 bits 30 / 25 / 38; 2,048 rows 4,096 x 4,096 64 x 128 / 128 x 128 / 128 x 256 / 256 x 256 bfloat16 72 / 64 / 59 / 87, 8 bits 67 / 59 / 58 / 91,
// 16,384 x 4,096 264 / 237 / 228 / 198, 250 / 227 / 222 / 199; 64 rows 4,096 x 4,096 2x1 / 4x1 / 2x4 12.8 / 10.6 / 10.8, 128 rows 2x1 / 2x4 / 4x4 22.8 / 10.6 / 16.4. Up to 16 rows the matrix's
// bytes set the pace: 16 waves a strip while every strip has a compute unit of its own (us, 16 waves / 8 waves on two strips: 1 row 1,600 x 6,400 5.0 / 6.7, 8
// rows 4,096 x 4,096 5.3 / 6.3, 1 row 4,096 x 16,384 9.7 / 13.6), two strips beyond (1 row 16,384 x 4,096 12.4 / 10.1, 8 rows 6,400 x 1,600 6.2 / 4.5).
// `same_bits`: eight waves whatever the rows, so that a row's sums have one order.
static int choose_shape(int kind, bool same_bits, int M, int N) {
    const int strips = mx_strips(N);
    if (M <= 16) return !same_bits && strips <= 256 ? kShape1x1 : kShape1x2;
    struct Shape {
        int id, rows, columns;
        float fixed[2], round[2];
    };
    static const Shape shapes[] = {
        {kShape2x1, 32, 16, {0, 0}, {7.6f, 7.0f}},       {kShape2x2, 32, 32, {0, 0}, {9.0f, 8.5f}},        {kShape4x1, 64, 16, {0, 0}, {9.7f, 9.7f}},
        {kShape2x4, 32, 64, {0, 0}, {10.6f, 11.0f}},     {kShape4x2, 64, 32, {0, 0}, {12.1f, 12.4f}},      {kShape4x4, 64, 64, {0, 0}, {16.4f, 16.8f}},
        {kMxTile64, 64, 128, {12.0f, 10.0f}, {15.3f, 13.9f}}, {kMxTile128, 128, 128, {10.5f, 12.0f}, {27.3f, 26.4f}}, {kMxTileWide, 128, 256, {0, 1.0f}, {55.5f, 55.3f}},
        {kMxTile256, 256, 256, {0, 0}, {92.0f, 95.0f}},
    };
    int best = kShape4x4;
    float least = 3e38f;
    for (const Shape& s : shapes) {
        if (s.id < 10 && (same_bits || M <= 64)) continue;
        const int64_t groups = (static_cast<int64_t>(M) + s.rows - 1) / s.rows * ((N + s.columns - 1) / s.columns);
        const float us = s.fixed[kind == kRowsMx] + static_cast<float>((groups + 255) / 256) * s.round[kind == kRowsMx];
        if (us < least) least = us, best = s.id;
    }
    return best;
}

template <int ROWS>
static int product_of_shape(int shape, const MxRowsIn& in, const uint8_t* blocks, int M, int N, int K, const EpiParams& epi, hipStream_t stream) {
    if constexpr (ROWS == kRowsF32) {  // (eight waves whatever the rows: every sum has one order)
        if (M <= 16) return launch_product<ROWS, 1, 1, 2, 8>(in, blocks, M, N, K, epi, stream);
        return launch_product<ROWS, 2, 1, 1, 8>(in, blocks, M, N, K, epi, stream);
    } else {
        switch (shape) {
            case kShape1x1: return launch_product<ROWS, 1, 1, 2, 16>(in, blocks, M, N, K, epi, stream);
            case kShape1x2: return launch_product<ROWS, 1, 2, 2, 8>(in, blocks, M, N, K, epi, stream);
            case kShape2x1: return launch_product<ROWS, 2, 1, 2, 8>(in, blocks, M, N, K, epi, stream);
            case kShape2x2: return launch_product<ROWS, 2, 2, 2, 8>(in, blocks, M, N, K, epi, stream);
            case kShape2x4: return launch_product<ROWS, 2, 4, 1, 8>(in, blocks, M, N, K, epi, stream);
            case kShape4x1: return launch_product<ROWS, 4, 1, 1, 8>(in, blocks, M, N, K, epi, stream);
            case kShape4x2: return launch_product<ROWS, 4, 2, 1, 8>(in, blocks, M, N, K, epi, stream);
            case kShape4x4: return launch_product<ROWS, 4, 4, 1, 8>(in, blocks, M, N, K, epi, stream);
            case kMxTile64:
            case kMxTile128:
            case kMxTileWide:
            case kMxTile256: return launch_mx_tiles(ROWS, shape, in, blocks, M, N, K, epi, stream);
            default: return fail(1, "mx_product: unknown shape %d", shape);
        }
    }
}

}  // namespace liyab

using namespace liyab;

// a: rows [M, lda] of `rows` 0: bfloat16, 1: float32, 2: e4m3 codes (padded with zeros to whole chunks) with their scales [M, lds].
// shape: 0 chooses from the sizes, -1 among those that leave a row the same bits whatever the other rows, a positive number is one of the shapes above.
extern "C" int liyab_mx_product(const void* a, int64_t lda, const void* a_scales, int64_t lds, int rows, const void* blocks, int M, int N, int K, int shape,
                                const EpiParams* epi, hipStream_t stream) {
    LIYAB_REQUIRE(a && blocks && epi, "mx_product: null pointer");
    LIYAB_REQUIRE(M >= 0 && N > 0 && K > 0, "mx_product: bad sizes");
    if (M == 0) return 0;
    if (const int rc = check_epilogue(*epi, M, N)) return rc;
    LIYAB_REQUIRE(epi->out_dtype == kF32 || epi->out_dtype == kBF16, "mx_product: unknown output dtype %d", epi->out_dtype);
    LIYAB_REQUIRE(reinterpret_cast<uintptr_t>(a) % 16 == 0 && reinterpret_cast<uintptr_t>(blocks) % 16 == 0, "mx_product: operands start on 16-byte boundaries");
    const MxRowsIn in{a, lda, static_cast<const uint8_t*>(a_scales), lds};
    const uint8_t* const b = static_cast<const uint8_t*>(blocks);
    if (shape == 0 && (lda >= (int64_t{1} << 22) || K >= (1 << 22))) shape = -1;  // (a tile's rows are found by 32-bit offsets)
    if (rows == kRowsMx) {
        LIYAB_REQUIRE(reinterpret_cast<uintptr_t>(a_scales) % 4 == 0, "mx_product: scales start on 4-byte boundaries");  // (a load into LDS takes four)
        LIYAB_REQUIRE(a_scales && lda >= static_cast<int64_t>(mx_chunks(K)) * kMxChunk && lda % 16 == 0 && lds >= mx_chunks(K) * 4, "mx_product: rows in 8 bits are padded to %d codes",
                      mx_chunks(K) * kMxChunk);
        return product_of_shape<kRowsMx>(shape > 0 ? shape : choose_shape(rows, shape < 0, M, N), in, b, M, N, K, *epi, stream);
    }
    const int per = rows == kRowsBF16 ? 8 : 4;
    LIYAB_REQUIRE(rows == kRowsBF16 || rows == kRowsF32, "mx_product: unknown kind of rows %d", rows);
    LIYAB_REQUIRE(K % per == 0 && lda % per == 0 && lda >= K, "mx_product: rows of whole pieces of 16 bytes are taken (K = %d, row stride %lld)", K, static_cast<long long>(lda));
    if (rows == kRowsF32) return product_of_shape<kRowsF32>(0, in, b, M, N, K, *epi, stream);
    return product_of_shape<kRowsBF16>(shape > 0 ? shape : choose_shape(rows, shape < 0, M, N), in, b, M, N, K, *epi, stream);
}
