// out[M, N] = rows[M, K] . matrix[N, K]^T for many rows, the matrix in 4 bits (mx.h), the rows in bfloat16 or 8 bits: a tile of the output a workgroup.
//
// Everything comes into LDS by direct loads, through a ring of three stages of 128 bytes a row (64 k of bfloat16, 128 of 8 bits) with the matrix blocks'
// numbers and scales that meet them; a stage is waited for by the count of the loads behind it, with one barrier, and the two stages after it stay in
// flight. Blocks lie in LDS as in memory, which is the order of the matrix instructions' operands; of a row the 16-byte piece p sits at position p ^ (row / 2 % 8), so that
// 16 lanes' reads of 16 rows at one piece fall into different banks.
//   bfloat16  a block's numbers become bfloat16 with their scale, two an instruction (exact), and meet 16x16x32 instructions
//   8 bits    the rows' numbers become bfloat16 too on their way from LDS (three bits of mantissa and a power of two: exact), then as above: sums of 32
//             bits, as wide rows have them. The scaled instruction (v_mfma_scale_f32_16x16x128_f8f6f4) would take both operands as they are at twice the rate, but it adds
//             eight neighbouring products in a sum of their own, in which the bits below 2^-13 of the largest are cut off (measured: 2^-14 of it is lost, 2^-13 is not):
//             5e-6 in the 2-norm over normal values, and all of what is left where large neighbours cancel. It took 118 us where this takes 199 (2,048 x 16,384 x 4,096).
// What bounds it: the matrix instructions at 256 x 256 (2,048 x 16,384 x 4,096, no activation: 198 us with rows in bfloat16, 1,390 TFLOP/s, and 199 in 8 bits; 8,192 cubed 1,430 TFLOP/s
// both, where a library product of bfloat16 matrices reaches 1,359); at the smaller tiles the instructions around them (2,048 x 4,096 x 4,096 at 128 x 256, one round of
// 256 workgroups: 59 and 58 us; 512 rows at 64 x 128: 29 and 25, the narrower rows being half the bytes). Measured on the way, us at 2,048 x
// 16,384 x 4,096 / 512 x 4,096 x 4,096 with the scaled instruction: loads' places worked out in each stage 119 / 21, kept in registers 116 / 17, the loads and the next stage's
// blocks spread over the steps 112 / 17, the reads' places as constants of the instructions 112 / 15.7. Six stages in place of three change nothing.
#include "common.h"
#include "gemm_tile.h"
#include "launchers.h"
#include "mx.h"
#include "mx_product.h"
#include "ring.h"

#include <atomic>

namespace liyab {

typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;

constexpr int kStageBytes = 128;  // of a row
constexpr int kTileStages = 3;

// A stage in LDS: the rows, the blocks' numbers, the blocks' scales (whole loads of 1 KB), the rows' scales (8 bits).
template <int ROWS, int BM, int BN>
struct MxStage {
    static constexpr int K = ROWS == kRowsMx ? kMxChunk : kMxChunk / 2;      // k
    static constexpr int BLOCK = 16 * K / 2, SCALES = 16 * K / kMxGroup;     // bytes of a strip's numbers and scales
    static constexpr int CODES_AT = BM * kStageBytes, SCALES_AT = CODES_AT + BN / 16 * BLOCK, ROW_SCALES_AT = SCALES_AT + 1024;
    static constexpr int BYTES = ROW_SCALES_AT + (ROWS == kRowsMx ? BM * 4 : 0);
};

template <int ROWS, int WM, int WN, int TM, int TN, typename OutT, int EPI>
__global__ void __launch_bounds__(64 * WM * WN)
mx_tile_kernel(MxRowsIn in, const uint8_t* __restrict__ blocks, int M, int N, int K, EpiParams epi, int vec_ok, int page_shift) {
    constexpr bool MX = ROWS == kRowsMx;
    constexpr int WAVES = WM * WN, BM = WM * TM * 16, BN = WN * TN * 16, STRIPS = BN / 16;
    using Stage = MxStage<ROWS, BM, BN>;
    constexpr int ROW_LOADS = BM / 8 / WAVES, CODE_LOADS = STRIPS * Stage::BLOCK / 1024 / WAVES, LOADS = ROW_LOADS + CODE_LOADS + 1;  // a wave and stage
    static_assert(ROW_LOADS * WAVES * 8 == BM && CODE_LOADS * WAVES * 1024 == STRIPS * Stage::BLOCK && BM / 64 <= WAVES / 2 && LOADS * (kTileStages - 1) <= 63, "a stage's loads");
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int wm = wave / WN, wn = wave % WN;
    const int g = lane / 16, r = lane % 16;
    int m0, n0;
    tile_place<BM, BN>(M, N, K, m0, n0);
    const int chunks = mx_chunks(K), last_strip = mx_strips(N) - 1 - n0 / 16, stages = (K + Stage::K - 1) / Stage::K;

    // The loads' places: a 32-bit offset a lane from the tile's own corner (the launcher sees to it that it fits), the same in every stage, and a base that
    // moves with the stages. Worked out anew for each stage they cost a wave some hundred instructions, with few products to hide them behind.
    // Rows past M and strips past N: the last ones again, not stored.
    const uint32_t stride = static_cast<uint32_t>(in.lda) * (MX ? 1 : 2), strip_bytes = static_cast<uint32_t>(chunks) * kMxBlockBytes;
    const uint8_t* const rows = static_cast<const uint8_t*>(in.a) + static_cast<int64_t>(m0) * stride;
    const uint8_t* const matrix = blocks + static_cast<int64_t>(n0 / 16) * strip_bytes;
    const int last = M - 1 - m0;
    uint32_t row_at[ROW_LOADS], code_at[CODE_LOADS], scale_at;
#pragma unroll
    for (int i = 0; i < ROW_LOADS; ++i) {
        const int row = (wave * ROW_LOADS + i) * 8 + lane / 8;
        row_at[i] = static_cast<uint32_t>(min(row, last)) * stride + ((lane % 8) ^ ((row >> 1) & 7)) * 16;
    }
#pragma unroll
    for (int i = 0; i < CODE_LOADS; ++i) {
        constexpr int LANES = Stage::BLOCK / 16;  // a strip's
        const int piece = (wave * CODE_LOADS + i) * 64 + lane, strip = piece / LANES;
        code_at[i] = static_cast<uint32_t>(min(strip, last_strip)) * strip_bytes + piece % LANES * 16;
    }
    const bool rows_scales = MX && wave < BM / 64;  // one load a wave: the first waves bring 64 rows' scales each (8 bits), the others all the strips'
    if (rows_scales) {
        scale_at = static_cast<uint32_t>(min(wave * 64 + lane, last)) * static_cast<uint32_t>(in.lds);
    } else {
        constexpr int PIECES = Stage::SCALES / 16;
        scale_at = static_cast<uint32_t>(min(min(lane / PIECES, STRIPS - 1), last_strip)) * strip_bytes + 1024 + lane % PIECES * 16;
    }
    const int tail = MX ? 0 : K % Stage::K * 2;  // bytes of a row in the last stage, if they don't fill it (rows in 8 bits are padded): zeros behind them
    auto issue = [&](int stage, uint8_t* to, auto load) {  // one load of a stage
        constexpr int i = decltype(load)::value, c = i - ROW_LOADS;
        const uint32_t s = static_cast<uint32_t>(min(stage, stages - 1));  // (past the end the last one again, into a place that nobody reads: the waits count on as many loads a stage)
        if constexpr (i < ROW_LOADS) {
            const int r0 = (wave * ROW_LOADS + i) * 8;
            const uint8_t* src = rows + static_cast<uint64_t>(s) * kStageBytes + row_at[i];
            if constexpr (!MX) {
                const bool beyond = ((lane % 8) ^ (((r0 + lane / 8) >> 1) & 7)) * 16 >= tail;
                if (tail != 0 && s == static_cast<uint32_t>(stages - 1) && beyond) src = reinterpret_cast<const uint8_t*>(mx_zeros());
            }
            __builtin_amdgcn_global_load_lds(src, (lds_void_ptr)(to + r0 * kStageBytes), 16, 0, 0);
            return;
        }
        // the stage's part of a block: all of it, or in bfloat16 one half of its k, which is half of its lanes
        const uint32_t chunk = MX ? s : s / 2, half = MX ? 0 : s % 2;
        if constexpr (i >= ROW_LOADS && i < LOADS - 1) {
            const uint8_t* const src = matrix + (chunk * kMxBlockBytes + half * Stage::BLOCK) + code_at[c];
            __builtin_amdgcn_global_load_lds(src, (lds_void_ptr)(to + Stage::CODES_AT + (wave * CODE_LOADS + c) * 1024), 16, 0, 0);
        } else if (rows_scales) {
            const uint8_t* const src = in.scales + m0 * in.lds + s * 4 + scale_at;
            __builtin_amdgcn_global_load_lds(src, (lds_void_ptr)(to + Stage::ROW_SCALES_AT + wave * 256), 4, 0, 0);
        } else {
            const uint8_t* const src = matrix + (chunk * kMxBlockBytes + half * Stage::SCALES) + scale_at;
            __builtin_amdgcn_global_load_lds(src, (lds_void_ptr)(to + Stage::SCALES_AT), 16, 0, 0);
        }
    };

    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // A stage is PHASES runs through the tile's rows, TM steps of TN products each; a phase multiplies eight of every lane's k. A step's row operand comes from
    // LDS AHEAD steps before it, also across stages: AHEAD steps before a stage's end everyone waits until the next one has arrived and this one has been read,
    // and the loads of the third stage from here take its place.
    // (Vectors of the compiler's own throughout: its reads of structs from LDS wait for every load into LDS.)
    constexpr int PHASES = MX ? 4 : 2, STEPS = TM * PHASES, AHEAD = 4;
    static_assert(STEPS % AHEAD == 0, "the operands' places are constants");
    struct Operand {
        u32x4 wide;      // eight k of bfloat16
        u32x2 codes;     // or of 8 bits
        uint32_t scale;  // and their group's byte
    };
    Operand ring[AHEAD];
    // (what a lane adds to a stage's place: everything else is a constant of the instruction)
    const int place = (r >> 1) & 7;  // (a tile's rows start at a multiple of 16)
    const int row_lane = (wm * TM * 16 + r) * kStageBytes, piece0 = row_lane + ((2 * g) ^ place) * 16, piece1 = row_lane + ((2 * g + 1) ^ place) * 16;
    const int row_scale_lane = Stage::ROW_SCALES_AT + (wm * TM * 16 + r) * 4 + g;
    const int code_lane = Stage::CODES_AT + wn * TN * Stage::BLOCK + (MX ? 16 * lane : (16 * (g / 2) + r) * 16 + g % 2 * 8);
    const int scale_lane = Stage::SCALES_AT + wn * TN * Stage::SCALES + (MX ? lane : 16 * (g / 2) + r);
    auto read = [&](Operand& x, const uint8_t* stage, int q) {
        const int i = q % TM, k = q / TM;
        if constexpr (MX) {
            x.codes = *reinterpret_cast<const u32x2*>(stage + (k < 2 ? piece0 : piece1) + k % 2 * 8 + i * 16 * kStageBytes);
            x.scale = stage[row_scale_lane + i * 16 * 4];
        } else {
            x.wide = *reinterpret_cast<const u32x4*>(stage + (k == 0 ? piece0 : piece1) + i * 16 * kStageBytes);
        }
    };
    // A stage's blocks: of a lane's matrix rows 32 k (8 bits: lane group g takes k 32 g .. 32 g + 31 of the 128), or 16 k of the half (bfloat16: k 16 g .. 16 g + 15 of the 64).
    using Codes = std::conditional_t<MX, u32x4, u32x2>;
    struct Blocks {
        Codes codes[TN];
        uint32_t scale[TN];
    };
    auto read_block = [&](Blocks& b, const uint8_t* stage, int j) {
        b.codes[j] = *reinterpret_cast<const Codes*>(stage + code_lane + j * Stage::BLOCK);
        b.scale[j] = stage[scale_lane + j * Stage::SCALES];
    };
    // eight k of the blocks as operands: those that are multiplied now, and those of the next phase
    mx_bf16x8 w[TN], w_next[TN];
    Blocks now, next;

    uint8_t *here = lds, *after = lds + Stage::BYTES;
#pragma unroll
    for (int s = 0; s < kTileStages; ++s) in_turn(std::make_integer_sequence<int, LOADS>{}, [&](auto load) { issue(s, lds + s * Stage::BYTES, load); });
    wait_loads<(kTileStages - 1) * LOADS>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int j = 0; j < TN; ++j) read_block(now, here, j);
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) read(ring[q], here, q);
#pragma unroll
    for (int j = 0; j < TN; ++j) w[j] = mx_eight_of(now.codes[j][0], mx_power(now.scale[j]));
    auto multiply = [&](Blocks& now, Blocks& next, int s) {
#pragma unroll
        for (int j = 0; j < TN; ++j) asm volatile("" : "+v"(now.scale[j]));  // (whole registers: bytes, they would be made so, and waited for, in the stage before)
        in_turn(std::make_integer_sequence<int, STEPS>{}, [&](auto at) {
            constexpr int q = decltype(at)::value, i = q % TM, k = q / TM;
            Operand& x = ring[q % AHEAD];
            mx_bf16x8 rows8;
            if constexpr (MX) rows8 = mx_eight_of_rows(x.codes[0], x.codes[1], mx_power(x.scale));
            else rows8 = __builtin_bit_cast(mx_bf16x8, x.wide);
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[j], rows8, acc[i][j], 0, 0, 0);
            if constexpr (k < PHASES - 1) {
#pragma unroll
                for (int j = 0; j < TN; ++j)
                    if (j * TM / TN == i) w_next[j] = mx_eight_of(now.codes[j][k + 1], mx_power(now.scale[j]));
            } else if constexpr (q >= STEPS - 2) {
#pragma unroll
                for (int j = 0; j < TN; ++j)
                    if (j / (TN / 2) == q - (STEPS - 2)) w_next[j] = mx_eight_of(next.codes[j][0], mx_power(next.scale[j]));
            }
            if constexpr (i == TM - 1) {
#pragma unroll
                for (int j = 0; j < TN; ++j) w[j] = w_next[j];
            }
            if constexpr (q == STEPS - AHEAD) {  // (behind the step's products, which hide the wait for the last reads)
#pragma unroll
                for (int j = 0; j < TN; ++j) asm volatile("" : "+v"(acc[i][j]));
                __builtin_amdgcn_sched_barrier(0);
                __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
                wait_loads<(kTileStages - 2) * LOADS>();
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
            }
            // The next stage's blocks and the loads of the third from here, spread over the steps: a wave issues them between its products.
            if constexpr (q >= STEPS - AHEAD) {
                constexpr int part = q - (STEPS - AHEAD), blocks_in = AHEAD / 2;
                if constexpr (part < blocks_in) {
#pragma unroll
                    for (int j = part * TN / blocks_in; j < (part + 1) * TN / blocks_in; ++j) read_block(next, after, j);
                }
                constexpr int from = part * LOADS / AHEAD;
                in_turn(std::make_integer_sequence<int, (part + 1) * LOADS / AHEAD - from>{},
                        [&](auto load) { issue(s + kTileStages, here, std::integral_constant<int, from + decltype(load)::value>{}); });
            }
            // (the products stay in their step: gathered behind the reads of a whole stage they would need its operands in registers at once)
#pragma unroll
            for (int j = 0; j < TN; ++j) asm volatile("" : "+v"(acc[i][j]));
            if constexpr (q + AHEAD < STEPS) read(x, here, q + AHEAD);
            else read(x, after, q + AHEAD - STEPS);
            __builtin_amdgcn_sched_barrier(0);
        });
        here = after;
        after = after == lds + (kTileStages - 1) * Stage::BYTES ? lds : after + Stage::BYTES;
    };
    for (int s = 0; s < stages; s += 2) {
        multiply(now, next, s);
        if (s + 1 < stages) multiply(next, now, s + 1);
    }
    wait_loads<0>();  // the stages' places become the store's
    lds_barrier();
    store_tile<BM, BN, OutT, EPI, WM, WN>(acc, reinterpret_cast<bf16_t*>(lds), epi, PartsParams{}, m0, n0, M, N, vec_ok, page_shift, wave, wm, wn, lane);
}

template <int ROWS, int WM, int WN, int TM, int TN, typename OutT, int EPI>
static int launch_tile(const MxRowsIn& in, const uint8_t* blocks, int M, int N, int K, const EpiParams& epi, hipStream_t stream) {
    constexpr int BM = WM * TM * 16, BN = WN * TN * 16;
    constexpr size_t RING = kTileStages * MxStage<ROWS, BM, BN>::BYTES, STAGING = staging_bytes<BM, BN, WM, WN, 1>(sizeof(OutT));
    constexpr size_t LDS = RING > STAGING ? RING : STAGING;
    static_assert(LDS <= 160 * 1024, "LDS");
    const int64_t tiles = static_cast<int64_t>((M + BM - 1) / BM) * ((N + BN - 1) / BN);
    LIYAB_REQUIRE(in.lda < (int64_t{1} << 22) && in.lds < (int64_t{1} << 22) && K < (1 << 22), "mx_product: rows of %lld values and K = %d are too long", static_cast<long long>(in.lda), K);
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

template <int ROWS>
static int tile_of_size(int tile, const MxRowsIn& in, const uint8_t* blocks, int M, int N, int K, const EpiParams& epi, hipStream_t stream) {
    switch (tile) {
        case kMxTile64: return tile_of_epilogue<ROWS, 2, 2, 2, 4>(in, blocks, M, N, K, epi, stream);
        case kMxTileWide: return tile_of_epilogue<ROWS, 2, 4, 4, 4>(in, blocks, M, N, K, epi, stream);
        case kMxTile128: return tile_of_epilogue<ROWS, 2, 2, 4, 4>(in, blocks, M, N, K, epi, stream);
        default: return tile_of_epilogue<ROWS, 2, 4, 8, 4>(in, blocks, M, N, K, epi, stream);
    }
}

int launch_mx_tiles(int kind, int tile, const MxRowsIn& in, const uint8_t* blocks, int M, int N, int K, const EpiParams& epi, hipStream_t stream) {
    return kind == kRowsMx ? tile_of_size<kRowsMx>(tile, in, blocks, M, N, K, epi, stream) : tile_of_size<kRowsBF16>(tile, in, blocks, M, N, K, epi, stream);
}

}  // namespace liyab
