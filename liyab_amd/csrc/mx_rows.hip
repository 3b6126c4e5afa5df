// Rows in 8 bits (mx.h), as products of 4-bit matrices read them: plain rows, a norm of the residual stream with a sublayer's result added
// to it, and the gate between a feed-forward's products.
//
// A lane takes eight neighbours, so that a group of 32 is a quad of lanes: its largest magnitude is two exchanges in the lanes' own data
// path, codes leave as 8 bytes a lane, the scale as one byte a quad. Rows of codes are padded to whole chunks of 128 k, with zeros,
// for the products' loads.
#include "activations.h"
#include "common.h"
#include "launchers.h"
#include "mx.h"

namespace liyab {

constexpr int kRowThreads = 256;
constexpr int kLaneValues = 8;

__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0xB1, 0xf, 0xf, false)));  // lane ^ 1
    return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x4E, 0xf, 0xf, false)));  // lane ^ 2
}

// Eight neighbours p[i .. i + 8), zeros from d on. WIDE: every row starts on a 16-byte boundary.
template <bool WIDE, typename T>
__device__ __forceinline__ void load8(float (&v)[kLaneValues], const T* p, int i, int d) {
    if (WIDE && i + kLaneValues <= d) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = *reinterpret_cast<const float4*>(p + i), b = *reinterpret_cast<const float4*>(p + i + 4);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 a = *reinterpret_cast<const uint4*>(p + i);
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[2 * j] = __uint_as_float(w[j] << 16);
                v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < kLaneValues; ++j) v[j] = i + j < d ? to_float<T>(p[i + j]) : 0.0f;
}

// Eight neighbours' codes and their group's scale to a row's places.
__device__ __forceinline__ void store_group(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int i, const float (&v)[kLaneValues]) {
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < kLaneValues; ++j) amax = max(amax, mx_magnitude(v[j]));
    const uint32_t s = mx_scale(quad_max(amax), kE4m3Max);
    *reinterpret_cast<uint2*>(codes + i) = mx_e4m3(v, s);
    if (threadIdx.x % 4 == 0) scales[i / kMxGroup] = static_cast<uint8_t>(s);
}

enum : int { kMxPlain = 0, kMxSilu = 1, kMxGeluTanh = 2, kMxClamped = 3 };

// Values next to a border of the 8-bit numbers, or of a group's scale, need more than 32 bits to fall on the right side: gates and norms are
// computed in 64 (whose multiply-adds go at the rate of single 32-bit ones) and come to 32 rounded to odd, which no later rounding is misled by. In 32 bits
// throughout some values of every 16 million landed on the wrong side, off by 1e-5 to 1e-4 in the 2-norm, now none (2,048 rows of 16,384: gates 54.5 us then
// and 54.6 now, 5.5 TB/s; norms of 2,048 rows of 4,096 19.7 and 20.5, 4.5 TB/s).
__device__ __forceinline__ float to_odd(double v) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = static_cast<uint32_t>(bits);
    // 29 bits more than 32-bit numbers have: whether there is any becomes the last bit
    const uint32_t cut = (lo | ((lo & 0x1fffffffu) + 0x1fffffffu)) & 0xe0000000u;
    return static_cast<float>(__builtin_bit_cast(double, (bits & 0xffffffff00000000ull) | cut));
}

// g / (1 + 2^t). 2^r for |r| <= 1/2: the polynomial of degree 7 that meets it at the eight Chebyshev points, off by 6e-11 of it.
__device__ __forceinline__ double over_one_plus(double g, double t) {
    const double n = rint(t), r = t - n;
    double e = 1.5303699899644103e-05;
    e = fma(e, r, 0.00015469729234889767);
    e = fma(e, r, 0.0013333478477891695);
    e = fma(e, r, 0.009618025613220747);
    e = fma(e, r, 0.05550410906319735);
    e = fma(e, r, 0.240226512134995);
    e = fma(e, r, 0.6931471805568348);
    e = fma(e, r, 0.9999999999595616);
    const double d = fmin(1.0 + __builtin_amdgcn_ldexp(e, static_cast<int>(n)), 1e300);  // (finite: an infinity's reciprocal could not be mended)
    const double rcp = __builtin_amdgcn_rcp(d);
    return g * fma(fma(-d, rcp, 1.0), rcp, rcp);
}
__device__ __forceinline__ double silu(double g) { return over_one_plus(g, -1.44269504088896340736 * g); }
__device__ __forceinline__ double gelu_tanh_of(double g) {
    constexpr double kSlope = -2.0 * 0.79788456080286535588 * 1.44269504088896340736;
    return over_one_plus(g, g * fma(kSlope * 0.044715, g * g, kSlope));
}

template <typename T, int OP, bool WIDE>
__global__ void __launch_bounds__(kRowThreads)
mx_rows_kernel(uint8_t* __restrict__ codes, int64_t ldo, uint8_t* __restrict__ scales, int64_t lds, const T* __restrict__ in, int64_t ldi, int d, int blocks_a_row,
               double limit, double slope, double shift) {
    const int64_t row = blockIdx.x / blocks_a_row;
    const int i = (blockIdx.x % blocks_a_row * kRowThreads + threadIdx.x) * kLaneValues;
    if (i >= ldo) return;  // (whole quads: rows of codes are whole chunks)
    const T* const p = in + row * ldi;
    float v[kLaneValues];
    load8<WIDE>(v, p, i, d);
    if constexpr (OP != kMxPlain) {
        float u[kLaneValues];
        load8<WIDE>(u, p + d, i, d);
#pragma unroll
        for (int j = 0; j < kLaneValues; ++j) {
            if constexpr (OP == kMxSilu) v[j] = to_odd(silu(v[j]) * u[j]);
            else if constexpr (OP == kMxGeluTanh) v[j] = to_odd(gelu_tanh_of(v[j]) * u[j]);
            else {
                // (comparisons, which leave NaN what it is)
                const double g = v[j] > limit ? limit : v[j], c = u[j] > limit ? limit : u[j] < -limit ? -limit : u[j];
                v[j] = to_odd(over_one_plus(g, -1.44269504088896340736 * slope * g) * (c + shift));
            }
            if (i + j >= d) v[j] = 0.0f;  // (behind the row)
        }
    }
    store_group(codes + row * ldo, scales + row * lds, i, v);
}

template <int CTRL>
__device__ __forceinline__ double double_dpp(double v) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(bits), CTRL, 0xf, 0xf, false), hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(bits >> 32), CTRL, 0xf, 0xf, false);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double double_of(double v, int lane) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(bits), lane), hi = __builtin_amdgcn_readlane(static_cast<int>(bits >> 32), lane);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

// The sum over a workgroup of WAVES waves, the same bits in every lane (the steps of `wave_sum`).
template <int WAVES>
__device__ __forceinline__ double group_total(double v, double* red) {
    v += double_dpp<0xB1>(v);
    v += double_dpp<0x4E>(v);
    v += double_dpp<0x141>(v);
    v += double_dpp<0x140>(v);
    v = (double_of(v, 0) + double_of(v, 16)) + (double_of(v, 32) + double_of(v, 48));
    if constexpr (WAVES > 1) {
        __syncthreads();
        if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = v;
        __syncthreads();
        v = 0.0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v += red[w];
    }
    return v;
}

// v scale weight + bias of eight neighbours, in 8 bits.
template <bool WIDE>
__device__ __forceinline__ void store_normed(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, double (&v)[kLaneValues], double scale, const float* __restrict__ weight,
                                             const float* __restrict__ bias, int i, int d) {
    float w[kLaneValues], b[kLaneValues] = {}, y[kLaneValues];
    if (weight != nullptr) {
        load8<WIDE>(w, weight, i, d);
#pragma unroll
        for (int j = 0; j < kLaneValues; ++j) v[j] *= scale * w[j];
    } else {
#pragma unroll
        for (int j = 0; j < kLaneValues; ++j) v[j] *= scale;
    }
    if (bias != nullptr) load8<WIDE>(b, bias, i, d);
#pragma unroll
    for (int j = 0; j < kLaneValues; ++j) y[j] = to_odd(v[j] + b[j]);
    if (i + kLaneValues > d) {  // (a row of infinities has NaN behind its end too)
#pragma unroll
        for (int j = 0; j < kLaneValues; ++j)
            if (i + j >= d) y[j] = 0.0f;
    }
    store_group(codes, scales, i, y);
}

// A row a workgroup, held in registers: TRIPS stretches of 8 values a lane. The stream may be x: a lane loads all that it stores before it stores.
template <int WAVES, int TRIPS, typename AddT, bool WIDE>
__global__ void __launch_bounds__(WAVES * kWave)
mx_norm_kernel(uint8_t* __restrict__ codes, int64_t ldo, uint8_t* __restrict__ scales, int64_t lds, const float* x, const AddT* add,
               float* stream, const float* __restrict__ weight, const float* __restrict__ bias, double eps, int centred, int d) {
    __shared__ double red[WAVES];
    constexpr int STEP = WAVES * kWave * kLaneValues;
    const int64_t row = blockIdx.x;
    const int i0 = threadIdx.x * kLaneValues;
    double v[TRIPS][kLaneValues], sum = 0.0;
#pragma unroll
    for (int t = 0; t < TRIPS; ++t) {
        float a[kLaneValues], y[kLaneValues] = {};
        load8<WIDE>(a, x + row * d, i0 + t * STEP, d);
        if (add != nullptr) load8<WIDE>(y, add + row * d, i0 + t * STEP, d);
#pragma unroll
        for (int j = 0; j < kLaneValues; ++j) v[t][j] = static_cast<double>(a[j]) + y[j];
    }
    if (stream != nullptr) {
        float* const s = stream + row * d;
#pragma unroll
        for (int t = 0; t < TRIPS; ++t) {
            const int i = i0 + t * STEP;
            if (WIDE && i + kLaneValues <= d) {
                *reinterpret_cast<float4*>(s + i) = make_float4(static_cast<float>(v[t][0]), static_cast<float>(v[t][1]), static_cast<float>(v[t][2]), static_cast<float>(v[t][3]));
                *reinterpret_cast<float4*>(s + i + 4) = make_float4(static_cast<float>(v[t][4]), static_cast<float>(v[t][5]), static_cast<float>(v[t][6]), static_cast<float>(v[t][7]));
            } else {
#pragma unroll
                for (int j = 0; j < kLaneValues; ++j)
                    if (i + j < d) s[i + j] = static_cast<float>(v[t][j]);
            }
        }
    }
    double mean = 0.0;
    if (centred) {
#pragma unroll
        for (int t = 0; t < TRIPS; ++t)
#pragma unroll
            for (int j = 0; j < kLaneValues; ++j) sum += v[t][j];
        mean = group_total<WAVES>(sum, red) / d;
        sum = 0.0;
    }
#pragma unroll
    for (int t = 0; t < TRIPS; ++t)
#pragma unroll
        for (int j = 0; j < kLaneValues; ++j) {
            v[t][j] = i0 + t * STEP + j < d ? v[t][j] - mean : 0.0;
            sum += v[t][j] * v[t][j];
        }
    const double scale = 1.0 / sqrt(group_total<WAVES>(sum, red) / d + eps);
#pragma unroll
    for (int t = 0; t < TRIPS; ++t) {
        const int i = i0 + t * STEP;
        if (i >= ldo) continue;
        store_normed<WIDE>(codes + row * ldo, scales + row * lds, v[t], scale, weight, bias, i, d);
    }
}

// Rows that registers do not hold: read again for the squares and for the result, each time as x + add, whose 64 bits the stream does not have. The stream
// may be x: it is written with the result, by the lane that reads there.
template <int WAVES, typename AddT, bool WIDE>
__global__ void __launch_bounds__(WAVES * kWave)
mx_norm_long_kernel(uint8_t* __restrict__ codes, int64_t ldo, uint8_t* __restrict__ scales, int64_t lds, const float* x, const AddT* add, float* stream,
                    const float* __restrict__ weight, const float* __restrict__ bias, double eps, int centred, int d) {
    __shared__ double red[WAVES];
    constexpr int STEP = WAVES * kWave * kLaneValues;
    const int64_t row = blockIdx.x;
    const int i0 = threadIdx.x * kLaneValues;
    auto values = [&](double (&v)[kLaneValues], int i) {
        float a[kLaneValues], y[kLaneValues] = {};
        load8<WIDE>(a, x + row * d, i, d);
        if (add != nullptr) load8<WIDE>(y, add + row * d, i, d);
#pragma unroll
        for (int j = 0; j < kLaneValues; ++j) v[j] = static_cast<double>(a[j]) + y[j];
    };
    double v[kLaneValues], sum = 0.0, mean = 0.0;
    if (centred) {
        for (int i = i0; i < d; i += STEP) {
            values(v, i);
#pragma unroll
            for (int j = 0; j < kLaneValues; ++j) sum += v[j];
        }
        mean = group_total<WAVES>(sum, red) / d;
    }
    sum = 0.0;
    for (int i = i0; i < d; i += STEP) {
        values(v, i);
#pragma unroll
        for (int j = 0; j < kLaneValues; ++j) {
            const double c = i + j < d ? v[j] - mean : 0.0;
            sum += c * c;
        }
    }
    const double scale = 1.0 / sqrt(group_total<WAVES>(sum, red) / d + eps);
    for (int i = i0; i < ldo; i += STEP) {
        values(v, i);
#pragma unroll
        for (int j = 0; j < kLaneValues; ++j) {
            if (stream != nullptr && i + j < d) stream[row * d + i + j] = static_cast<float>(v[j]);
            v[j] -= mean;
        }
        store_normed<WIDE>(codes + row * ldo, scales + row * lds, v, scale, weight, bias, i, d);
    }
}

// Rows of 2- or 4-byte values as the products load them: whole pieces of 16 bytes, zeros behind the row.
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
mx_align_kernel(T* __restrict__ out, int ldo, const T* __restrict__ in, int64_t ldi, int d, int blocks_a_row) {
    const int64_t row = blockIdx.x / blocks_a_row;
    const int i = blockIdx.x % blocks_a_row * kRowThreads + threadIdx.x;
    if (i < ldo) out[row * ldo + i] = i < d ? in[row * ldi + i] : T(0);
}

static bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// The places of n rows of d values in 8 bits.
static int check_rows(const char* what, const void* codes, int64_t ldo, const void* scales, int64_t lds, int n, int d) {
    LIYAB_REQUIRE(codes && scales, "%s: null pointer", what);
    LIYAB_REQUIRE(n >= 0 && d > 0, "%s: bad sizes", what);
    LIYAB_REQUIRE(ldo == static_cast<int64_t>(mx_chunks(d)) * kMxChunk && lds >= ldo / kMxGroup && reinterpret_cast<uintptr_t>(codes) % 8 == 0,
                  "%s: rows of %d values take %d codes a row (got %lld) and as many scales as groups", what, d, mx_chunks(d) * kMxChunk, static_cast<long long>(ldo));
    return 0;
}

template <typename T, int OP>
static int launch_rows(const char* what, void* codes, int64_t ldo, void* scales, int64_t lds, const void* in, int64_t ldi, int n, int d, double limit, double slope,
                       double shift, hipStream_t stream) {
    const int per_row = static_cast<int>((ldo / kLaneValues + kRowThreads - 1) / kRowThreads);
    const int64_t grid = static_cast<int64_t>(n) * per_row;
    LIYAB_REQUIRE(grid < (int64_t{1} << 31), "%s: %d rows of %d values are too many", what, n, d);
    constexpr int per16 = 16 / sizeof(T);
    const bool wide = aligned16(in) && ldi % per16 == 0 && (OP == kMxPlain || d % per16 == 0);
    auto* kernel = wide ? &mx_rows_kernel<T, OP, true> : &mx_rows_kernel<T, OP, false>;
    kernel<<<static_cast<unsigned>(grid), kRowThreads, 0, stream>>>(static_cast<uint8_t*>(codes), ldo, static_cast<uint8_t*>(scales), lds, static_cast<const T*>(in), ldi,
                                                                    d, per_row, limit, slope, shift);
    return check_launch(what);
}

struct NormArgs {
    void *codes, *scales;
    int64_t ldo, lds;
    const float* x;
    const void* add;
    float* stream_out;
    const float *weight, *bias;
    double eps;
    int centred, n, d;
    hipStream_t stream;
};

template <int WAVES, int TRIPS, typename AddT>
static int launch_norm(const NormArgs& a, bool wide) {
    auto* kernel = wide ? &mx_norm_kernel<WAVES, TRIPS, AddT, true> : &mx_norm_kernel<WAVES, TRIPS, AddT, false>;
    kernel<<<a.n, WAVES * kWave, 0, a.stream>>>(static_cast<uint8_t*>(a.codes), a.ldo, static_cast<uint8_t*>(a.scales), a.lds, a.x, static_cast<const AddT*>(a.add),
                                                a.stream_out, a.weight, a.bias, a.eps, a.centred, a.d);
    return check_launch("mx_norm");
}

template <typename AddT>
static int norm_of_width(const NormArgs& a, bool wide) {
    if (a.d <= 512) return launch_norm<1, 1, AddT>(a, wide);
    if (a.d <= 2048) return launch_norm<4, 1, AddT>(a, wide);
    if (a.d <= 4096) return launch_norm<4, 2, AddT>(a, wide);
    if (a.d <= 8192) return launch_norm<8, 2, AddT>(a, wide);
    if (a.d <= 16384) return launch_norm<16, 2, AddT>(a, wide);
    auto* kernel = wide ? &mx_norm_long_kernel<16, AddT, true> : &mx_norm_long_kernel<16, AddT, false>;
    kernel<<<a.n, 16 * kWave, 0, a.stream>>>(static_cast<uint8_t*>(a.codes), a.ldo, static_cast<uint8_t*>(a.scales), a.lds, a.x, static_cast<const AddT*>(a.add),
                                             a.stream_out, a.weight, a.bias, a.eps, a.centred, a.d);
    return check_launch("mx_norm");
}

}  // namespace liyab

using namespace liyab;

extern "C" int liyab_mx_rows(void* codes, int64_t ldo, void* scales, int64_t lds, const void* x, int dtype, int64_t ldx, int n, int d, hipStream_t stream) {
    if (const int rc = check_rows("mx_rows", codes, ldo, scales, lds, n, d)) return rc;
    LIYAB_REQUIRE(x != nullptr && ldx >= d, "mx_rows: needs rows of %d values", d);
    if (n == 0) return 0;
    if (dtype == kF32) return launch_rows<float, kMxPlain>("mx_rows", codes, ldo, scales, lds, x, ldx, n, d, 0, 0, 0, stream);
    if (dtype == kBF16) return launch_rows<bf16_t, kMxPlain>("mx_rows", codes, ldo, scales, lds, x, ldx, n, d, 0, 0, 0, stream);
    return fail(1, "mx_rows: unknown dtype %d", dtype);
}

// act 0: silu, 1: the tanh form of gelu, 2: clamped halves (limit, slope, shift).
extern "C" int liyab_mx_glu(void* codes, int64_t ldo, void* scales, int64_t lds, const float* gu, int64_t ld, int n, int d, int act, double limit, double slope,
                            double shift, hipStream_t stream) {
    if (const int rc = check_rows("mx_glu", codes, ldo, scales, lds, n, d)) return rc;
    LIYAB_REQUIRE(gu != nullptr && ld >= 2 * static_cast<int64_t>(d), "mx_glu: needs rows of 2 x %d values", d);
    LIYAB_REQUIRE(act != 2 || limit > 0.0, "mx_glu: the limit must be positive");
    if (n == 0) return 0;
    if (act == 0) return launch_rows<float, kMxSilu>("mx_glu", codes, ldo, scales, lds, gu, ld, n, d, 0, 0, 0, stream);
    if (act == 1) return launch_rows<float, kMxGeluTanh>("mx_glu", codes, ldo, scales, lds, gu, ld, n, d, 0, 0, 0, stream);
    if (act == 2) return launch_rows<float, kMxClamped>("mx_glu", codes, ldo, scales, lds, gu, ld, n, d, limit, slope, shift, stream);
    return fail(1, "mx_glu: unknown activation %d", act);
}

extern "C" int liyab_mx_norm(void* codes, int64_t ldo, void* scales, int64_t lds, const float* x, const void* add, int add_dtype, float* stream_out,
                             const float* weight, const float* bias, double eps, int centred, int n, int d, hipStream_t stream) {
    if (const int rc = check_rows("mx_norm", codes, ldo, scales, lds, n, d)) return rc;
    LIYAB_REQUIRE(x != nullptr && d <= 65536, "mx_norm: needs rows of up to 65,536 values, got %d", d);
    if (n == 0) return 0;
    const NormArgs a{codes, scales, ldo, lds, x, add, stream_out, weight, bias, eps, centred != 0, n, d, stream};
    const int per16 = add != nullptr && add_dtype == kBF16 ? 8 : 4;
    const bool wide = d % per16 == 0 && aligned16(x) && aligned16(add) && aligned16(stream_out) && aligned16(weight) && aligned16(bias);
    if (add_dtype == kF32) return norm_of_width<float>(a, wide);
    if (add_dtype == kBF16) return norm_of_width<bf16_t>(a, wide);
    return fail(1, "mx_norm: unknown dtype %d", add_dtype);
}

// out [n, ldo] = in [n, ldi]'s first d values of `size` bytes, zeros behind them; ldo up to a piece of 16 bytes more than d.
extern "C" int liyab_mx_align(void* out, int ldo, const void* in, int64_t ldi, int size, int n, int d, hipStream_t stream) {
    LIYAB_REQUIRE(out && in, "mx_align: null pointer");
    LIYAB_REQUIRE(n >= 0 && d > 0 && ldo >= d && ldi >= d && (size == 2 || size == 4), "mx_align: bad sizes");
    const int per_row = (ldo + kRowThreads - 1) / kRowThreads;
    const int64_t grid = static_cast<int64_t>(n) * per_row;
    LIYAB_REQUIRE(grid < (int64_t{1} << 31), "mx_align: %d rows of %d values are too many", n, d);
    if (n == 0) return 0;
    if (size == 2) mx_align_kernel<uint16_t><<<static_cast<unsigned>(grid), kRowThreads, 0, stream>>>(static_cast<uint16_t*>(out), ldo, static_cast<const uint16_t*>(in), ldi, d, per_row);
    else mx_align_kernel<uint32_t><<<static_cast<unsigned>(grid), kRowThreads, 0, stream>>>(static_cast<uint32_t*>(out), ldo, static_cast<const uint32_t*>(in), ldi, d, per_row);
    return check_launch("mx_align");
}
