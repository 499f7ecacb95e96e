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

template <class T>
struct Raw8 {  // eight values as they lie
    typedef T vec __attribute__((ext_vector_type(8)));
    typedef T any __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    vec v;
    __device__ __forceinline__ float operator[](int e) const { return (float)v[e]; }
};
// Eight values' nearest whole numbers to 127 x / most, a byte each.  x * inv is off by less than 2^-16 (two roundings of a
// value up to 127), so it decides alone except next to a half, where the difference from the quotient is taken without error: of
// 127 x and n most the rounding errors are kept, and their difference and that to most / 2 are of close numbers.
// Adding 1.5 x 2^23 rounds to a whole number, whose two's complement is then the sum's low byte.
template <class T>
__device__ __forceinline__ uint2 quantized8(const Raw8<T> &x, const RowScale &r) {
    if (r.inv == 0.f) return make_uint2(0, 0);
    constexpr float kRound = 0x1.8p23f;
    uint32_t t[8];
    float far = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float y = x[e] * r.inv, s = y + kRound;
        far = fmaxf(far, fabsf(y - (s - kRound)));
        t[e] = __float_as_uint(s);
    }
    if (__builtin_expect(far > 0.5f - 0x1p-15f, 0)) {
        const float most = r.most * 0x1p-8f, half = 0.5f * most;  // 127 x stays finite
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int n = (int)(int8_t)t[e];
            const float w = x[e] * 0x1p-8f, p = w * 127.f, q = (float)n * most;
            const float d = p - q, low = fmaf(w, 127.f, -p) - fmaf((float)n, most, -q);
            const float over = d > 0 ? (d - half) + low : (-d - half) - low;  // |127 x - n most| - most / 2, or its sign
            if (over > 0 || (over == 0 && (n & 1))) t[e] = (uint32_t)(n + (d > 0 ? 1 : -1));
        }
    }
    const auto four = [](uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
        const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0C0C0400), hi = __builtin_amdgcn_perm(d, c, 0x0C0C0400);
        return lo | hi << 16;
    };
    return make_uint2(four(t[0], t[1], t[2], t[3]), four(t[4], t[5], t[6], t[7]));
}
template <class T>
__device__ __forceinline__ uint32_t magnitude(const Raw8<T> &x) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) m = max(m, __float_as_uint(x[e]) & 0x7FFFFFFFu);
    return m;
}
// Up to eight values of a row from d on, 0 beyond its end.  UNIT: they lie on end, and are read 16 bytes at a time wherever they
// start.
template <bool UNIT, class T>
__device__ __forceinline__ Raw8<T> row8(const T *row, int64_t ds, int d, int dim) {
    Raw8<T> x;
    if (UNIT && d + 8 <= dim) {
        x.v = *reinterpret_cast<const typename Raw8<T>::any *>(row + d);
    } else {
        const T *p = row + (UNIT ? d : d * ds);
#pragma unroll
        for (int e = 0; e < 8; e++) x.v[e] = d + e < dim ? p[UNIT ? e : e * ds] : (T)0.f;
    }
    return x;
}

// A row's values d = 512 c + 8 lane .. + 7, c < HOLD
template <int HOLD, class T>
struct RowStart {
    Raw8<T> x[HOLD];
};
template <bool UNIT, int HOLD, class T>
__device__ __forceinline__ RowStart<HOLD, T> row_start(const T *row, const Source &s, int lane) {
    RowStart<HOLD, T> r;
#pragma unroll
    for (int c = 0; c < HOLD; c++) r.x[c] = row8<UNIT>(row, s.sd, c * 512 + lane * 8, s.dim);
    return r;
}
// A row by one wave: put(d, bytes) takes values d .. d + 7, zeros from dim to dimp (a multiple of 8); returns the scale.  Rows of up
// to 512 HOLD values are read once, by row_start; the rest of longer ones twice.
template <bool UNIT, int HOLD, class T, class Put>
__device__ __forceinline__ float quantize_row(const T *row, const RowStart<HOLD, T> &start, const Source &s, int dimp, int lane, Put &&put) {
    uint32_t most = 0;
#pragma unroll
    for (int c = 0; c < HOLD; c++) most = max(most, magnitude(start.x[c]));
#pragma unroll 2
    for (int d = HOLD * 512 + lane * 8; d < s.dim; d += 512) most = max(most, magnitude(row8<UNIT>(row, s.sd, d, s.dim)));
    const RowScale r = row_scale(gs_wave_max_u32(most));
#pragma unroll
    for (int c = 0; c < HOLD; c++)
        if (c * 512 + lane * 8 < dimp) put(c * 512 + lane * 8, quantized8(start.x[c], r));
#pragma unroll 1
    for (int d = HOLD * 512 + lane * 8; d < dimp; d += 512) put(d, quantized8(row8<UNIT>(row, s.sd, d, s.dim), r));
    return r.scale;
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

// A column's scale and bias
struct ColumnScale {
    float by, bias;
};
__device__ __forceinline__ ColumnScale column_scale(int v, const Weight8 &W, const void *bias, int type) {
    return v < W.n ? ColumnScale{W.scales[v], bias_at(bias, type, v)} : ColumnScale{0.f, 0.f};
}

// Products of at most 64 rows, their values on end, in one launch, for latency: a workgroup of eight waves quantises all rows into
// LDS itself and takes blocks of 16 columns, KS of its waves a block, each its part of k.  The weight goes from memory to the
// operands' registers: a lane takes 32 bytes on end of its column, so that a wave's loads take whole lines, and the first of them
// are asked for before the rows are quantised.  What bounds it is the weight's bytes and latency: one row of 768 values, 30522
// columns 6.4 us (3.7 TB/s), 24 rows 13 (in two launches 14); one row of 1024, 4096 columns 5.
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
    ColumnScale next;  // of the lane's column
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
        next = epi.column(c0 + i, W);
    };

    // The wave's rows, every eighth (those that are left out are not read).  The first kRows are asked for before the weight, whose
    // loads would have to land before theirs otherwise (24 rows, 30522 columns of 768: 12.5 -> 11.5 us).
    const auto here = [&](int r) { return r < rows && ((kept >> r) & 1); };
    const auto quantize = [&](int r, const RowStart<2, T> &x) {
        const float scale = quantize_row<true, 2>(source_row<T>(h, r), x, h, kp, lane,
                                                  [&](int d, uint2 y) { *reinterpret_cast<uint2 *>(smem + r * ls + d) = y; });
        if (lane == 0) scales[r] = scale * kDown;
    };
    constexpr int kRows = MB > 2 ? 4 : 2 * MB;
    {
        RowStart<2, T> x[kRows];
#pragma unroll
        for (int u = 0; u < kRows; u++)
            if (here(wave + u * kFewWaves)) x[u] = row_start<true, 2>(source_row<T>(h, wave + u * kFewWaves), h, lane);
        __builtin_amdgcn_sched_barrier(0);
        seek();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < kRows; u++)
            if (here(wave + u * kFewWaves)) quantize(wave + u * kFewWaves, x[u]);
    }
    if (kRows * kFewWaves < 16 * MB)
        for (int r = wave + kRows * kFewWaves; r < rows; r += kFewWaves)
            if (here(r)) quantize(r, row_start<true, 2>(source_row<T>(h, r), h, lane));
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
        const ColumnScale col = next;
        g += gridDim.x;
        const bool more = g < groups;
        if (more) seek();
        if (KS == 1) {
            epi.template run<MB>(acc, done + i, W, col, scales, rows, kept, q);
        } else {
#pragma unroll
            for (int m = 0; m < MB; m++) part[(wave * MB + m) * 64 + lane] = acc[m];
            __syncthreads();
            if (wave == 0) {
#pragma unroll
                for (int m = 0; m < MB; m++)
#pragma unroll
                    for (int k = 1; k < kFewWaves; k++) acc[m] += part[(k * MB + m) * 64 + lane];
                epi.template run<MB>(acc, done + i, W, col, scales, rows, kept, q);
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

inline bool few8_ok(int rows, int kp, int64_t dim_stride) { return dim_stride == 1 && rows <= kFewRows && few_lds(rows, kp, kFewWaves) <= kFewLds; }

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
