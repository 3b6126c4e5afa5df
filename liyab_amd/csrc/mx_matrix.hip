// Matrices in 4 bits (mx.h): made of wide ones or of codes and scales in plain rows, and back. Run once a matrix, at load: a lane takes a
// group of 32, whose place in a block is its own.
#include "common.h"
#include "launchers.h"
#include "mx.h"

namespace liyab {

constexpr int kMatrixWaves = 4;

// The lane's group: block number, row and first k.
struct MxPlace {
    int64_t block;
    int64_t row;
    int k;
};
__device__ __forceinline__ MxPlace mx_place(int chunks) {
    const int lane = threadIdx.x % kWave;
    const int64_t block = static_cast<int64_t>(blockIdx.x) * kMatrixWaves + threadIdx.x / kWave;
    return {block, block / chunks * kMxStrip + lane % 16, static_cast<int>(block % chunks) * kMxChunk + lane / 16 * kMxGroup};
}

template <typename T>
__global__ void __launch_bounds__(kMatrixWaves * kWave)
mx_quantize_kernel(uint8_t* __restrict__ blocks, const T* __restrict__ w, int64_t ldw, int N, int K, int chunks, int64_t n_blocks) {
    const MxPlace at = mx_place(chunks);
    if (at.block >= n_blocks) return;
    float v[kMxGroup];
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < kMxGroup; ++i) {
        v[i] = at.row < N && at.k + i < K ? to_float<T>(w[at.row * ldw + at.k + i]) : 0.0f;
        amax = max(amax, mx_magnitude(v[i]));
    }
    const uint32_t s = mx_scale(amax, kE2m1Max);
    const float f = mx_factor(s);
    uint32_t out[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {  // (past 6 the conversion stays at 6)
        uint32_t c = 0;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * q + 0] * f, v[8 * q + 1] * f, 1.0f, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * q + 2] * f, v[8 * q + 3] * f, 1.0f, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * q + 4] * f, v[8 * q + 5] * f, 1.0f, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * q + 6] * f, v[8 * q + 7] * f, 1.0f, 3);
        out[q] = s == 255u ? 0u : c;
    }
    uint8_t* b = blocks + at.block * kMxBlockBytes;
    const int lane = threadIdx.x % kWave;
    *reinterpret_cast<uint4*>(b + 16 * lane) = make_uint4(out[0], out[1], out[2], out[3]);
    b[1024 + lane] = static_cast<uint8_t>(s);
}

__global__ void __launch_bounds__(kMatrixWaves * kWave)
mx_pack_kernel(uint8_t* __restrict__ blocks, const uint8_t* __restrict__ codes, int64_t ldc, const uint8_t* __restrict__ scales, int64_t lds,
               int N, int K, int chunks, int64_t n_blocks) {
    const MxPlace at = mx_place(chunks);
    if (at.block >= n_blocks) return;
    const bool inside = at.row < N && at.k < K;
    uint32_t out[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int k = at.k + 2 * i;
        uint32_t byte = inside && k < K ? codes[at.row * ldc + k / 2] : 0u;
        if (k + 1 >= K) byte &= 15u;  // an odd row's last byte
        out[i / 4] |= byte << (8 * (i % 4));
    }
    uint8_t* b = blocks + at.block * kMxBlockBytes;
    const int lane = threadIdx.x % kWave;
    *reinterpret_cast<uint4*>(b + 16 * lane) = make_uint4(out[0], out[1], out[2], out[3]);
    b[1024 + lane] = inside ? scales[at.row * lds + at.k / kMxGroup] : 0;
}

template <typename T>
__global__ void __launch_bounds__(kMatrixWaves * kWave)
mx_dense_kernel(T* __restrict__ w, int64_t ldw, const uint8_t* __restrict__ blocks, int N, int K, int chunks, int64_t n_blocks) {
    const MxPlace at = mx_place(chunks);
    if (at.block >= n_blocks || at.row >= N) return;
    const uint8_t* b = blocks + at.block * kMxBlockBytes;
    const int lane = threadIdx.x % kWave;
    const uint4 c = *reinterpret_cast<const uint4*>(b + 16 * lane);
    const float power = mx_power(b[1024 + lane]);
    const uint32_t word[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        mx_f32x2 v;
        switch (i % 4) {  // (the byte's number is part of the instruction)
            case 0: v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[i / 4], power, 0); break;
            case 1: v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[i / 4], power, 1); break;
            case 2: v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[i / 4], power, 2); break;
            default: v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[i / 4], power, 3); break;
        }
        const int k = at.k + 2 * i;
        if (k < K) w[at.row * ldw + k] = from_float<T>(v[0]);
        if (k + 1 < K) w[at.row * ldw + k + 1] = from_float<T>(v[1]);
    }
}

// The blocks of a matrix and the workgroups that take a wave each; 0 where they do not fit a grid.
static int64_t matrix_blocks(int N, int K) { return static_cast<int64_t>(mx_strips(N)) * mx_chunks(K); }
static unsigned matrix_grid(int64_t n_blocks) {
    const int64_t groups = (n_blocks + kMatrixWaves - 1) / kMatrixWaves;
    return groups < (int64_t{1} << 31) ? static_cast<unsigned>(groups) : 0u;
}

}  // namespace liyab

using namespace liyab;

extern "C" int liyab_mx_quantize(void* blocks, const void* w, int dtype, int64_t ldw, int N, int K, hipStream_t stream) {
    LIYAB_REQUIRE(blocks && w, "mx_quantize: null pointer");
    LIYAB_REQUIRE(N > 0 && K > 0 && ldw >= K, "mx_quantize: bad sizes");
    const int64_t nb = matrix_blocks(N, K);
    const unsigned grid = matrix_grid(nb);
    LIYAB_REQUIRE(grid > 0, "mx_quantize: a matrix of %d x %d is too large", N, K);
    uint8_t* out = static_cast<uint8_t*>(blocks);
    if (dtype == kF32) mx_quantize_kernel<float><<<grid, kMatrixWaves * kWave, 0, stream>>>(out, static_cast<const float*>(w), ldw, N, K, mx_chunks(K), nb);
    else if (dtype == kBF16) mx_quantize_kernel<bf16_t><<<grid, kMatrixWaves * kWave, 0, stream>>>(out, static_cast<const bf16_t*>(w), ldw, N, K, mx_chunks(K), nb);
    else return fail(1, "mx_quantize: unknown dtype %d", dtype);
    return check_launch("mx_quantize");
}

extern "C" int liyab_mx_pack(void* blocks, const void* codes, int64_t ldc, const void* scales, int64_t lds, int N, int K, hipStream_t stream) {
    LIYAB_REQUIRE(blocks && codes && scales, "mx_pack: null pointer");
    LIYAB_REQUIRE(N > 0 && K > 0 && ldc >= (K + 1) / 2 && lds >= (K + kMxGroup - 1) / kMxGroup, "mx_pack: bad sizes");
    const int64_t nb = matrix_blocks(N, K);
    const unsigned grid = matrix_grid(nb);
    LIYAB_REQUIRE(grid > 0, "mx_pack: a matrix of %d x %d is too large", N, K);
    mx_pack_kernel<<<grid, kMatrixWaves * kWave, 0, stream>>>(static_cast<uint8_t*>(blocks), static_cast<const uint8_t*>(codes), ldc,
                                                              static_cast<const uint8_t*>(scales), lds, N, K, mx_chunks(K), nb);
    return check_launch("mx_pack");
}

extern "C" int liyab_mx_dense(void* w, int dtype, int64_t ldw, const void* blocks, int N, int K, hipStream_t stream) {
    LIYAB_REQUIRE(w && blocks, "mx_dense: null pointer");
    LIYAB_REQUIRE(N > 0 && K > 0 && ldw >= K, "mx_dense: bad sizes");
    const int64_t nb = matrix_blocks(N, K);
    const unsigned grid = matrix_grid(nb);
    LIYAB_REQUIRE(grid > 0, "mx_dense: a matrix of %d x %d is too large", N, K);
    const uint8_t* in = static_cast<const uint8_t*>(blocks);
    if (dtype == kF32) mx_dense_kernel<float><<<grid, kMatrixWaves * kWave, 0, stream>>>(static_cast<float*>(w), ldw, in, N, K, mx_chunks(K), nb);
    else if (dtype == kBF16) mx_dense_kernel<bf16_t><<<grid, kMatrixWaves * kWave, 0, stream>>>(static_cast<bf16_t*>(w), ldw, in, N, K, mx_chunks(K), nb);
    else return fail(1, "mx_dense: unknown dtype %d", dtype);
    return check_launch("mx_dense");
}
