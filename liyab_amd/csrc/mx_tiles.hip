// out[M, N] = rows[M, K] . matrix[N, K]^T for many rows, the matrix in 4 bits (mx.h), the rows in bfloat16 or 8 bits: a tile of the output a workgroup.
//
// Only the rows go through LDS. The matrix lies in memory as the matrix instructions read it, 16 rows and 128 k a block, so each wave
// loads the blocks of its own columns into registers, one chunk of K ahead; the waves of a workgroup that share columns find them in the
// L1. Rows come into LDS by direct loads (16 bytes a lane), two stages of 256 bytes a row: 128 k of bfloat16 or 256 of 8 bits; one is
// multiplied while the other fills, and the loads are waited for once a stage. Within a row the 16-byte piece p sits at position p ^ (row % 16), so that
// 16 lanes' reads of 16 rows at one piece fall into different banks.
//   bfloat16  a block's numbers become bfloat16 with their scale, two an instruction (exact), and meet four 16x16x32 instructions
//   8 bits    one scaled 16x16x128 instruction a block takes both operands and both scales as they are, at twice bfloat16's rate. It adds eight
//             neighbouring products in a sum of their own, in which the bits below 2^-13 of the largest are cut off (measured: 2^-14 of it is lost,
//             2^-13 is not), and those sums in 32 bits: the result is off by 5e-6 in the 2-norm, a four-hundredth of a rounding to
//             bfloat16 and a five-thousandth of what rows in 8 bits are off from wider ones by. Up to 64 rows, where memory sets the pace, mx_product.hip
//             keeps 32 bits throughout.
#include "common.h"
#include "gemm_tile.h"
#include "launchers.h"
#include "mx.h"
#include "mx_product.h"

#include <atomic>

namespace liyab {

typedef __attribute__((address_space(3))) void* mx_lds_ptr;

constexpr int kStageBytes = 256;  // of a row

template <int ROWS, int WM, int WN, int TM, int TN, typename OutT, int EPI>
__global__ void __launch_bounds__(64 * WM * WN)
mx_tile_kernel(MxRowsIn in, const uint8_t* __restrict__ blocks, int M, int N, int K, EpiParams epi, int vec_ok, int page_shift) {
    constexpr int WAVES = WM * WN, BM = WM * TM * 16, BN = WN * TN * 16;
    constexpr int LOADS = BM / 4 / WAVES;                       // wave-loads of 4 rows a wave and stage
    constexpr int HALVES = ROWS == kRowsMx ? 2 : 1;             // chunks of 128 k a stage
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int wm = wave / WN, wn = wave % WN;
    const int g = lane / 16, r = lane % 16;
    int m0, n0;
    tile_place<BM, BN>(M, N, K, m0, n0);
    const int chunks = mx_chunks(K), strips = mx_strips(N), stages = (chunks + HALVES - 1) / HALVES;

    // this lane's part in a wave-load: a row of four and the position of a piece in it
    const int64_t row_bytes = ROWS == kRowsMx ? static_cast<int64_t>(chunks) * kMxChunk : 2 * static_cast<int64_t>(K);
    const int64_t stride = in.lda * (ROWS == kRowsMx ? 1 : 2);  // (under 2^23: what a lane adds to its tile's first row fits 32 bits)
    const uint8_t* const rows = static_cast<const uint8_t*>(in.a) + m0 * stride;
    const int last = M - 1 - m0;
    auto issue = [&](int s) {
        uint8_t* const to = lds + (s & 1) * (BM * kStageBytes);
        const uint8_t* const at = rows + static_cast<int64_t>(s) * kStageBytes;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int r0 = (wave * LOADS + i) * 4, row = r0 + lane / 16, piece = ((lane % 16) ^ (row & 15)) * 16;
            const uint8_t* src = at + (static_cast<uint32_t>(min(row, last)) * static_cast<uint32_t>(stride) + piece);
            if (static_cast<int64_t>(s) * kStageBytes + piece >= row_bytes) src = reinterpret_cast<const uint8_t*>(mx_zeros());
            __builtin_amdgcn_global_load_lds(src, (mx_lds_ptr)(to + r0 * kStageBytes), 16, 0, 0);
        }
    };

    const uint8_t* block[TN];  // (the same in every lane)
#pragma unroll
    for (int j = 0; j < TN; ++j) block[j] = blocks + static_cast<int64_t>(min(n0 / 16 + wn * TN + j, strips - 1)) * chunks * kMxBlockBytes;
    struct Blocks {
        uint4 codes[TN];
        uint32_t scale[TN];
    };
    const uint32_t lane16 = 16 * lane;
    auto fetch = [&](Blocks& b, int c) {
        const int64_t at = static_cast<int64_t>(min(c, chunks - 1)) * kMxBlockBytes;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const uint8_t* const p = block[j] + at;
            b.codes[j] = *reinterpret_cast<const uint4*>(p + lane16);
            b.scale[j] = p[1024 + static_cast<uint32_t>(lane)];
        }
    };
    const uint8_t* const scales = ROWS == kRowsMx ? in.scales + m0 * in.lds : nullptr;
    uint32_t scale_at[ROWS == kRowsMx ? TM : 1];
    if constexpr (ROWS == kRowsMx) {
#pragma unroll
        for (int i = 0; i < TM; ++i) scale_at[i] = static_cast<uint32_t>(min((wm * TM + i) * 16 + r, last)) * static_cast<uint32_t>(in.lds) + g;
    }

    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    issue(0);
    Blocks now, next;
    fetch(now, 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    for (int s = 0; s < stages; ++s) {
        if (s + 1 < stages) issue(s + 1);
        const uint8_t* const from = lds + (s & 1) * (BM * kStageBytes) + (wm * TM * 16 + r) * kStageBytes;
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
            const int c = s * HALVES + h;
            if (h > 0 && c >= chunks) break;  // (an odd chunk is the last)
            fetch(next, c + 1);
            if constexpr (ROWS == kRowsMx) {
                uint32_t rs[TM];
#pragma unroll
                for (int i = 0; i < TM; ++i) rs[i] = (scales + 4 * c)[scale_at[i]];
#pragma unroll
                for (int i = 0; i < TM; ++i) {
                    const uint4 lo = *reinterpret_cast<const uint4*>(from + i * 16 * kStageBytes + ((8 * h + g) ^ r) * 16);
                    const uint4 hi = *reinterpret_cast<const uint4*>(from + i * 16 * kStageBytes + ((8 * h + 4 + g) ^ r) * 16);
                    const mx_i32x8 x = {static_cast<int>(lo.x), static_cast<int>(lo.y), static_cast<int>(lo.z), static_cast<int>(lo.w),
                                        static_cast<int>(hi.x), static_cast<int>(hi.y), static_cast<int>(hi.z), static_cast<int>(hi.w)};
#pragma unroll
                    for (int j = 0; j < TN; ++j) {
                        const mx_i32x8 w = {static_cast<int>(now.codes[j].x), static_cast<int>(now.codes[j].y), static_cast<int>(now.codes[j].z),
                                            static_cast<int>(now.codes[j].w), 0, 0, 0, 0};
                        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, acc[i][j], 4, 0, 0, now.scale[j], 0, rs[i]);
                    }
                }
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    mx_bf16x8 w[TN];
#pragma unroll
                    for (int j = 0; j < TN; ++j) {
                        const uint32_t word = k == 0 ? now.codes[j].x : k == 1 ? now.codes[j].y : k == 2 ? now.codes[j].z : now.codes[j].w;
                        w[j] = mx_eight_of(word, mx_power(now.scale[j]));
                    }
#pragma unroll
                    for (int i = 0; i < TM; ++i) {
                        const mx_bf16x8 x = *reinterpret_cast<const mx_bf16x8*>(from + i * 16 * kStageBytes + ((4 * g + k) ^ r) * 16);
#pragma unroll
                        for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[j], x, acc[i][j], 0, 0, 0);
                    }
                }
            }
            now = next;
        }
        // the next stage has arrived, and everyone is done reading this one
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }
    store_tile<BM, BN, OutT, EPI, WM, WN>(acc, reinterpret_cast<bf16_t*>(lds), epi, PartsParams{}, m0, n0, M, N, vec_ok, page_shift, wave, wm, wn, lane);
}

template <int ROWS, int WM, int WN, int TM, int TN, typename OutT, int EPI>
static int launch_tile(const MxRowsIn& in, const uint8_t* blocks, int M, int N, int K, const EpiParams& epi, hipStream_t stream) {
    constexpr int BM = WM * TM * 16, BN = WN * TN * 16;
    constexpr size_t STAGES = 2 * BM * kStageBytes, STAGING = staging_bytes<BM, BN, WM, WN, 1>(sizeof(OutT));
    constexpr size_t LDS = STAGES > STAGING ? STAGES : STAGING;
    static_assert(LDS <= 160 * 1024, "LDS");
    const int64_t tiles = static_cast<int64_t>((M + BM - 1) / BM) * ((N + BN - 1) / BN);
    LIYAB_REQUIRE(in.lda < (int64_t{1} << 22), "mx_product: a row stride of %lld", static_cast<long long>(in.lda));
    LIYAB_REQUIRE(tiles < (int64_t{1} << 31), "mx_product: %d x %d outputs are too many", M, N);
    int vec_ok, page_shift;
    store_rules<OutT, EPI>(epi, N, vec_ok, page_shift);
    auto* kernel = &mx_tile_kernel<ROWS, WM, WN, TM, TN, OutT, EPI>;
    static std::atomic<bool> ready{false};  // once a kernel
    if (LDS > 64 * 1024 && !ready.load(std::memory_order_relaxed)) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (e != hipSuccess) return fail(2, "mx_product: %s", hipGetErrorString(e));
        ready.store(true, std::memory_order_relaxed);
    }
    kernel<<<static_cast<unsigned>(tiles), 64 * WM * WN, LDS, stream>>>(in, blocks, M, N, K, epi, vec_ok, page_shift);
    return check_launch("mx_product");
}

template <int ROWS, int WM, int WN, int TM, int TN>
static int tile_of_epilogue(const MxRowsIn& in, const uint8_t* blocks, int M, int N, int K, const EpiParams& epi, hipStream_t stream) {
    const bool half = epi.out_dtype == kBF16;
#define LIYAB_TILE(MODE) \
    (half ? launch_tile<ROWS, WM, WN, TM, TN, bf16_t, MODE>(in, blocks, M, N, K, epi, stream) : launch_tile<ROWS, WM, WN, TM, TN, float, MODE>(in, blocks, M, N, K, epi, stream))
    switch (epi.mode) {
        case kEpiGeluTanh: return LIYAB_TILE(kEpiGeluTanh);
        case kEpiGeluErf: return LIYAB_TILE(kEpiGeluErf);
        case kEpiQkvPaged: return LIYAB_TILE(kEpiQkvPaged);
        case kEpiResidual: return launch_tile<ROWS, WM, WN, TM, TN, float, kEpiResidual>(in, blocks, M, N, K, epi, stream);
        default: return LIYAB_TILE(kEpiNone);
    }
#undef LIYAB_TILE
}

int launch_mx_tiles(int kind, int tile, const MxRowsIn& in, const uint8_t* blocks, int M, int N, int K, const EpiParams& epi, hipStream_t stream) {
    if (kind == kRowsMx)
        return tile == kMxTile128 ? tile_of_epilogue<kRowsMx, 2, 2, 4, 4>(in, blocks, M, N, K, epi, stream) : tile_of_epilogue<kRowsMx, 2, 4, 8, 4>(in, blocks, M, N, K, epi, stream);
    return tile == kMxTile128 ? tile_of_epilogue<kRowsBF16, 2, 2, 4, 4>(in, blocks, M, N, K, epi, stream) : tile_of_epilogue<kRowsBF16, 2, 4, 8, 4>(in, blocks, M, N, K, epi, stream);
}

}  // namespace liyab
