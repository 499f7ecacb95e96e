// Rows in 8 bits, and products of few of them.
//
// A row x is kept as whole numbers q = the nearest to 127 x / max |x| (ties to even) and one scale, max |x| / 127 in fp32.
// What a product of such rows needs is exact until its end: sums of q_x q_w fit 32 bits (32768 x 128^2 = 2^29), and
//     l = (sum of q_x q_w) * scale_x * scale_w + bias
// takes one rounding of the sum to fp32, one per scale and one with the bias.  The scales of x are multiplied by 2^-24 where
// they are made and the 2^24 is part of the last fma: so neither factor overflows or falls below the normal range before
// l itself does (scales are 0 or 2^-101 to 2^121).
//
// A row with an infinity or a NaN has scale NaN, and everything made from it is NaN.  One whose largest magnitude is below
// 2^-94 counts as zeros.
#pragma once

#include "gs_vocab_gemm.h"

namespace gsv {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kPad8 = 128;              // rows are zero to a multiple of this
constexpr float kLeast8 = 0x1p-94f;     // rows of smaller magnitudes are zeros
constexpr float kDown = 0x1p-24f, kUp = 0x1p24f;

// An operand of k_product: pairs of 8-bit values in the place of 16-bit ones, so that a stage is 128 values of k, and its sums
// are bits of whole numbers.  (Which byte of a fragment is which k does not matter, as long as both operands agree.)
struct I8 {
    using store_t = int8_t;
    __device__ __forceinline__ static i32x4 mfma(i32x4 a, i32x4 b, i32x4 c) {
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
    }
    __device__ __forceinline__ static f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
        return __builtin_bit_cast(
            f32x4, mfma(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), __builtin_bit_cast(i32x4, c)));
    }
};

struct RowScale {
    float most, inv, scale;  // inv: 127 / most; 0 where all values are kept as 0
};
// bits: the largest of the values' bits without their signs, above infinity's where one is NaN
__device__ __forceinline__ RowScale row_scale(uint32_t bits) {
    RowScale r;
    r.most = __uint_as_float(bits);
    const bool none = bits >= 0x7F800000u || r.most < kLeast8;
    r.inv = none ? 0.f : 127.f / r.most;
    r.scale = bits >= 0x7F800000u ? __builtin_nanf("") : none ? 0.f : r.most / 127.f;
    return r;
}
// The nearest whole number to 127 x / most.  x * inv is off by less than 2^-15 (three roundings of a value up to 127), so it
// decides alone except next to a half, where the difference from the quotient is taken in 64 bits, without error: 127 x, n most
// and their difference are of fewer than 53 bits there.
__device__ __forceinline__ int quantized(float x, const RowScale &r) {
    if (r.inv == 0.f) return 0;
    const float y = x * r.inv;
    float n = rintf(y);
    if (__builtin_expect(fabsf(fabsf(y - n) - 0.5f) < 0x1p-10f, 0)) {
        const double off = fma(-(double)n, (double)r.most, (double)x * 127.0), half = 0.5 * (double)r.most;
        if (fabs(off) > half || (fabs(off) == half && ((int)n & 1))) n += off > 0 ? 1.f : -1.f;
    }
    return (int)n;
}
__device__ __forceinline__ uint32_t quantized4(f32x4 x, const RowScale &r) {
    return (quantized(x[0], r) & 255) | (quantized(x[1], r) & 255) << 8 | (quantized(x[2], r) & 255) << 16 |
           (uint32_t)quantized(x[3], r) << 24;
}
__device__ __forceinline__ uint32_t magnitude(f32x4 x) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) m = max(m, __float_as_uint(x[e]) & 0x7FFFFFFFu);
    return m;
}

// N rows by one wave: put(u, d, word) takes row u's values d .. d + 3, zeros from dim to dimp (a multiple of 4); returns the
// scales.  Rows of up to 256 HOLD values are read once, all at a time; longer ones twice.
template <int HOLD, int N, class T, class Put>
__device__ __forceinline__ void quantize_rows(const T *const (&row)[N], const Source &s, int dimp, int lane, float (&scale)[N],
                                              Put &&put) {
    f32x4 x[N][HOLD];
    uint32_t most[N];
#pragma unroll
    for (int u = 0; u < N; u++) {
#pragma unroll
        for (int c = 0; c < HOLD; c++) x[u][c] = row4(row[u], s.sd, c * 256 + lane * 4, s.dim, s.vec);
    }
#pragma unroll
    for (int u = 0; u < N; u++) {
        most[u] = 0;
#pragma unroll
        for (int c = 0; c < HOLD; c++) most[u] = max(most[u], magnitude(x[u][c]));
        for (int d = HOLD * 256 + lane * 4; d < s.dim; d += 256) most[u] = max(most[u], magnitude(row4(row[u], s.sd, d, s.dim, s.vec)));
    }
#pragma unroll
    for (int u = 0; u < N; u++) {
        const RowScale r = row_scale(gs_wave_max_u32(most[u]));
        scale[u] = r.scale;
#pragma unroll
        for (int c = 0; c < HOLD; c++)
            if (c * 256 + lane * 4 < dimp) put(u, c * 256 + lane * 4, quantized4(x[u][c], r));
        for (int d = HOLD * 256 + lane * 4; d < dimp; d += 256) put(u, d, quantized4(row4(row[u], s.sd, d, s.dim, s.vec), r));
    }
}

// The weight: rows of 8-bit values, and their scales.
struct Weight8 {
    const int8_t *p;
    int64_t stride;  // bytes, a multiple of kPad8
    const float *scales;
    int n;
};

__device__ __forceinline__ float bias_at(const void *bias, int type, int v) {
    if (!bias) return 0.f;
    return type == GS_H_F32 ? ((const float *)bias)[v]
                            : type == GS_H_F16 ? (float)((const _Float16 *)bias)[v] : (float)((const __bf16 *)bias)[v];
}

// Products of at most 64 rows in one launch, for latency: a workgroup of eight waves quantises all rows into LDS itself and
// takes blocks of 16 columns, KS of its waves a block, each its part of k.  The weight goes from memory to the operands'
// registers: a lane takes 32 bytes on end of its column, so that a wave's loads take whole lines, and the first of them are asked
// for before the rows are quantised.
constexpr int kFewRows = 64, kFewLds = 80 * 1024, kFewWaves = 8;

__host__ __device__ inline int few_stride(int kp) { return kp + 16; }  // rows start 4 banks apart
inline int few_blocks(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }  // of 16 rows, that k_few8 is made for
inline size_t few_lds(int rows, int kp, int ks) {
    const int blocks = few_blocks(rows);
    return (size_t)rows * few_stride(kp) + kFewRows * 4 + (ks > 1 ? (size_t)kFewWaves * blocks * 1024 : 0);
}

template <class T, int MB, int KS, class Epi>
__global__ __launch_bounds__(64 * kFewWaves, 2) void k_few8(Source h, const uint8_t *mask, int rows, Weight8 W, int kp, int groups, Epi epi) {
    static_assert(KS == 1 || KS == kFewWaves, "a wave of its own for each block of columns, or all of them for one");
    extern __shared__ __align__(1024) char smem[];
    const int lane = gs_lane(), wave = gs_uniform((int)threadIdx.x >> 6), i = lane & 15, q = lane >> 4;
    const int ls = few_stride(kp);
    float *scales = reinterpret_cast<float *>(smem + (size_t)rows * ls);
    i32x4 *part = reinterpret_cast<i32x4 *>(scales + kFewRows);
    const uint64_t kept = __ballot(lane < rows && (!mask || mask[min(lane, rows - 1)] != 0));
    const int steps = kp / kPad8, k0 = KS == 1 ? 0 : steps * wave / KS, k1 = KS == 1 ? steps : steps * (wave + 1) / KS;

    constexpr int kAhead = 4;  // steps of 128 values in each of two buffers
    i32x4 w[2][2 * kAhead];
    int g = blockIdx.x, c0;
    __amdgpu_buffer_rsrc_t from;
    const auto load = [&](i32x4 (&b)[2 * kAhead], int k) {
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            if (k + u >= k1) break;
#pragma unroll
            for (int e = 0; e < 2; e++)
                b[2 * u + e] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(from, (int)(i * W.stride) + q * 32 + e * 16,
                                                                                              (k + u) * kPad8, 0));
        }
    };
    const auto seek = [&]() {
        c0 = KS == 1 ? (g * kFewWaves + wave) * 16 : g * 16;
        const int n = max(0, min(16, W.n - c0));
        from = gs_rsrc(W.p + (int64_t)(n ? c0 : 0) * W.stride, (uint32_t)(n * (int)W.stride));
        load(w[0], k0);
        load(w[1], k0 + kAhead);
    };
    seek();

    for (int r = wave * 2; r < rows; r += 2 * kFewWaves) {
        const int second = min(r + 1, rows - 1);
        if (!((kept >> r | kept >> second) & 1)) continue;
        // a row that is left out is not read
        const int a = (kept >> r) & 1 ? r : second, b = (kept >> second) & 1 ? second : r;
        const T *const row[2] = {source_row<T>(h, a), source_row<T>(h, b)};
        const int at[2] = {a, b};
        float s[2];
        quantize_rows<3, 2>(row, h, kp, lane, s, [&](int u, int d, uint32_t x) { *reinterpret_cast<uint32_t *>(smem + at[u] * ls + d) = x; });
        if (lane == 0) scales[a] = s[0] * kDown, scales[b] = s[1] * kDown;
    }
    __syncthreads();

    while (true) {
        i32x4 acc[MB];
#pragma unroll
        for (int m = 0; m < MB; m++) acc[m] = i32x4{0, 0, 0, 0};
        const auto multiply = [&](const i32x4 (&b)[2 * kAhead], int k) {
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
                if (k + u >= k1) break;
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int m = 0; m < MB; m++) {
                        const int row = min(16 * m + i, rows - 1);  // those past the last are not looked at
                        const i32x4 a = *reinterpret_cast<const i32x4 *>(smem + row * ls + (k + u) * kPad8 + q * 32 + e * 16);
                        acc[m] = I8::mfma(a, b[2 * u + e], acc[m]);
                    }
            }
        };
        for (int k = k0; k < k1; k += 2 * kAhead) {
            multiply(w[0], k);
            load(w[0], k + 2 * kAhead);
            multiply(w[1], k + kAhead);
            load(w[1], k + 3 * kAhead);
        }
        const int done = c0;
        g += gridDim.x;
        const bool more = g < groups;
        if (more) seek();
        if (KS == 1) {
            epi.template run<MB>(acc, done + i, W, scales, rows, kept, q);
        } else {
#pragma unroll
            for (int m = 0; m < MB; m++) part[(wave * MB + m) * 64 + lane] = acc[m];
            __syncthreads();
            if (wave == 0) {
#pragma unroll
                for (int m = 0; m < MB; m++)
#pragma unroll
                    for (int k = 1; k < kFewWaves; k++) acc[m] += part[(k * MB + m) * 64 + lane];
                epi.template run<MB>(acc, done + i, W, scales, rows, kept, q);
            }
            __syncthreads();
        }
        if (!more) break;
    }
}

inline int cu_count(int *cus) {
    int dev = 0;
    GS_CHECK_HIP(hipGetDevice(&dev));
    GS_CHECK_HIP(hipDeviceGetAttribute(cus, hipDeviceAttributeMultiprocessorCount, dev));
    return GS_OK;
}

inline bool few8_ok(int rows, int kp) { return rows <= kFewRows && few_lds(rows, kp, kFewWaves) <= kFewLds; }

// Once per device and kernel: LDS beyond 64 KiB
inline int allow_lds(const void *f, int bytes, std::atomic<uint64_t> &set) {
    int dev = 0;
    GS_CHECK_HIP(hipGetDevice(&dev));
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (!(set.load(std::memory_order_relaxed) & bit)) {
        GS_CHECK_HIP(hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
        set.fetch_or(bit, std::memory_order_relaxed);
    }
    return GS_OK;
}

template <class T, int MB, int KS, class Epi>
int launch_few8(const Source &h, const uint8_t *mask, int rows, const Weight8 &W, int kp, const Epi &epi, int cus, hipStream_t s) {
    static std::atomic<uint64_t> set{0};
    if (int rc = allow_lds(reinterpret_cast<const void *>(&k_few8<T, MB, KS, Epi>), kFewLds, set)) return rc;
    const int columns = KS == 1 ? 16 * kFewWaves : 16, groups = (W.n + columns - 1) / columns;
    hipLaunchKernelGGL((k_few8<T, MB, KS, Epi>), dim3((unsigned)(groups < cus ? groups : cus)), dim3(64 * kFewWaves),
                       few_lds(rows, kp, KS), s, h, mask, rows, W, kp, groups, epi);
    GS_CHECK_LAUNCH();
    return GS_OK;
}
// A block of columns is shared by a workgroup's waves where there would be too few of them for the GPU otherwise.
template <class T, class Epi>
int launch_few8(const Source &h, const uint8_t *mask, int rows, const Weight8 &W, int kp, const Epi &epi, int cus, hipStream_t s) {
    const bool split = (int64_t)W.n < (int64_t)64 * cus;
#define GSV_FEW8(MB)                                                                  \
    return split ? launch_few8<T, MB, kFewWaves, Epi>(h, mask, rows, W, kp, epi, cus, s) \
                 : launch_few8<T, MB, 1, Epi>(h, mask, rows, W, kp, epi, cus, s)
    switch (few_blocks(rows)) {
        case 1: GSV_FEW8(1);
        case 2: GSV_FEW8(2);
        default: GSV_FEW8(4);
    }
#undef GSV_FEW8
}

}  // namespace gsv
