// Rows in 8 bits, and products of few of them.
//
// A row x is kept as whole numbers q = the nearest to 127 x / max |x| (ties to even) and one scale, max |x| / 127 in fp32.
// What a product of such rows needs is exact until its end: sums of q_x q_w fit 32 bits (32768 x 128^2 = 2^29), and
//     l = (sum of q_x q_w) * scale_x * scale_w + bias
// takes one rounding of the sum to fp32, one per scale and one with the bias.  The scales of x are multiplied by 2^-24 where
// they are made and the 2^24 is part of the last fma, so that nothing overflows before l itself does (scales are 0 or 2^-101 to
// 2^121).  Its price is at the other end: what the fma multiplies is l 2^-24, below the normal range where l (without its bias) is
// below 2^-102, and l is then off by up to 2^-126 more.
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
    float most, inv, scale;  // largest magnitude times 2^-8; 1 / that, 0 where all values are kept as 0
};
// bits: the largest of the values' bits without their signs, above infinity's where one is NaN
__device__ __forceinline__ RowScale row_scale(uint32_t bits) {
    const float most = __uint_as_float(bits);
    const bool odd = bits >= 0x7F800000u, none = odd || most < kLeast8;
    return {most * 0x1p-8f, none ? 0.f : __builtin_amdgcn_rcpf(most * 0x1p-8f), odd ? __builtin_nanf("") : none ? 0.f : most / 127.f};
}
template <class T>
struct Raw8 {  // eight values as they lie
    typedef T vec __attribute__((ext_vector_type(8)));
    typedef T any __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    vec v;
    __device__ __forceinline__ float operator[](int e) const { return (float)v[e]; }
};
// Eight values' nearest whole numbers to p / most (p = 127 x, both times 2^-8, so that p stays finite), a byte each.
//
// y = p inv is off by a few units; y + (p - y most) inv is the quotient to half a unit and, where that is n + 1/2, exactly that.
// 16-bit values: p has no rounding, and no other quotient is nearer to n + 1/2 than 2^-19 of itself (2 p and (2n + 1) most are both
// whole multiples of x's last place, 2 p of less than 254 x 2^11), far beyond y's error, so rounding y is rounding the
// quotient.  fp32: p's rounding error `low` is kept; where y is n + 1/2 the sign of p + low - y most, which is exact there, says on which
// side the quotient is.  Adding 1.5 x 2^23 rounds to the nearest whole number, ties to even, whose two's complement is then the
// sum's low byte.  (Deciding by x * inv alone except next to a half costs less, but the code for the halves, once for each place where
// rows are quantised, has to come from memory: 24 rows and 30522 columns of 768 12.9 us instead of 10.5.)
template <class T>
__device__ __forceinline__ uint2 quantized8(const Raw8<T> &x, const RowScale &r) {
    if (r.inv == 0.f) return make_uint2(0, 0);
    constexpr float kRound = 0x1.8p23f, kMul = 127.f * 0x1p-8f;
    uint32_t t[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float p = x[e] * kMul, y0 = p * r.inv;
        if constexpr (sizeof(T) == 2) {
            t[e] = __float_as_uint(fmaf(fmaf(-y0, r.most, p), r.inv, y0) + kRound);
        } else {
            const float low = fmaf(x[e], kMul, -p);
            const float y = fmaf(fmaf(-y0, r.most, p) + low, r.inv, y0), n = rintf(y);
            const float rest = fmaf(-y, r.most, p) + low;
            t[e] = __float_as_uint((fabsf(y - n) == 0.5f && rest != 0.f ? y + copysignf(0.5f, rest) : n) + kRound);
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

// A maximum over a text's rows is taken of their sums times their own scales, and the column's scale multiplies that alone: as its
// magnitude, since a scale below zero, which a weight made elsewhere may have, turns the order round, so that its column's
// values change sign first.  An infinite one makes a NaN of some values, which are maxima.  (Not of NaN scales: all values are NaN.)
__device__ __forceinline__ bool reorders(float by) { return by < 0.f || by == INFINITY; }
__device__ __forceinline__ float in_order(float x, const ColumnScale &c) {
    if (fabsf(c.by) == INFINITY) {
        const float l = fmaf(x * c.by, kUp, c.bias);
        if (l != l) return l;
    }
    return c.by < 0.f ? -x : x;
}

// Products of at most 128 rows, their values on end, in one launch, for latency: a workgroup of eight waves quantises all rows into
// LDS itself and takes blocks of 16 columns, KS of its waves a block, each its part of k.  The weight goes from memory to the
// operands' registers: a lane takes 32 bytes on end of its column, so that a wave's loads take whole lines, and the first of them
// are asked for before the rows are quantised.  What bounds it is the weight's bytes and latency: one row of 768 values, 30522
// columns 6.3 us (3.7 TB/s), 24 rows 10.5; one row of 1024, 4096 columns 4.  How many rows fit LDS depends on their width (few8_ok, which
// asks for both ways of sharing columns): 128 of up to 512 values for term weights, 100 of 768, 75 of 1024; 32 of up to 4096 for linear layers.
constexpr int kFewRows = 128, kFewWaves = 8, kFewLds = 150 * 1024;
constexpr int kFewPitch = 17;  // of a row of 16 values that an epilogue leaves in LDS

// Rows that count, a bit each
struct Kept {
    uint64_t lo, hi;
    __device__ __forceinline__ bool operator()(int r) const { return (r < 64 ? lo >> r : hi >> (r - 64)) & 1; }
};

__host__ __device__ inline int few_stride(int kp) { return kp + 16; }  // rows start 4 banks apart
inline int few_blocks(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : rows <= 64 ? 4 : 8; }  // of 16 rows, that k_few8 is made for
// joins: whether the epilogue passes values through LDS
inline size_t few_lds(int rows, int kp, int ks, bool joins) {
    const size_t blocks = few_blocks(rows), values = blocks * 16 * kFewPitch * 4;
    return (size_t)rows * few_stride(kp) + kFewRows * 4 + (ks > 1 ? kFewWaves * blocks * 1024 + values : joins ? kFewWaves * values : 0);
}

template <class T, int MB, int KS, class Epi>
__global__ __launch_bounds__(64 * kFewWaves, 2) void k_few8(Source h, const uint8_t *mask, int rows, Weight8 W, int kp, int groups, Epi epi) {
    static_assert(KS == 1 || KS == kFewWaves, "a wave of its own for each block of columns, or all of them for one");
    extern __shared__ __align__(1024) char smem[];
    const int lane = gs_lane(), wave = gs_uniform((int)threadIdx.x >> 6), i = lane & 15, q = lane >> 4;
    const int ls = few_stride(kp);
    float *scales = reinterpret_cast<float *>(smem + (size_t)rows * ls);
    i32x4 *part = reinterpret_cast<i32x4 *>(scales + kFewRows);
    constexpr int values = MB * 16 * kFewPitch;  // KS > 1: one set, after the parts; else a wave's own
    float *left = reinterpret_cast<float *>(part) + (KS > 1 ? kFewWaves * MB * 256 : wave * values);
    const auto ballot = [&](int r) { return __ballot(r < rows && (!mask || mask[min(r, rows - 1)] != 0)); };
    const Kept kept{ballot(lane), MB > 4 ? ballot(lane + 64) : 0};
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
    // loads would have to land before theirs otherwise (24 rows, 30522 columns of 768: a microsecond).
    const auto here = [&](int r) { return r < rows && kept(r); };
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
#pragma unroll
            for (int m = 0; m < MB; m++) epi.block(acc[m], m, done + i, W, col, scales, rows, lane, left);
            if (Epi::joins) {
                gs_wave_sync();
                epi.finish(left, done + i, W, col, kept, lane, 0, 1);
                gs_wave_sync();
            }
        } else {
#pragma unroll
            for (int m = 0; m < MB; m++) part[(wave * MB + m) * 64 + lane] = acc[m];
            __syncthreads();
            if (wave < MB) {  // a wave joins the parts of a block of rows
                i32x4 sum = part[wave * 64 + lane];
#pragma unroll
                for (int k = 1; k < kFewWaves; k++) sum += part[(k * MB + wave) * 64 + lane];
                epi.block(sum, wave, done + i, W, col, scales, rows, lane, left);
            }
            __syncthreads();
            if (Epi::joins) epi.finish(left, done + i, W, col, kept, lane, wave, kFewWaves);
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

template <class Epi>
bool few8_ok(int rows, int kp, int64_t dim_stride) {
    return dim_stride == 1 && rows <= Epi::most_rows && few_lds(rows, kp, kFewWaves, Epi::joins) <= kFewLds && few_lds(rows, kp, 1, Epi::joins) <= kFewLds;
}

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
                       few_lds(rows, kp, KS, Epi::joins), s, h, mask, rows, W, kp, groups, epi);
    GS_CHECK_LAUNCH();
    return GS_OK;
}
// A block of columns is shared by a workgroup's waves where there would be too few of them for the GPU otherwise, below 16384 columns on
// 256 CUs.  us, shared and not:
//   columns                     1024        8192       12288       16384       20480       30522
//   linear, 1 x 768         3.7   5.5   4.6   5.8   5.4   5.8   6.2   5.9   7.0   5.9   9.5   5.9
//   1 x 1024                3.7   6.2   4.7   6.4   5.4   6.5   6.3   6.5   7.1   6.7  10.0   6.8
//   32 x 768                8.1  10.5   9.6  10.9  10.7  11.0  11.9  11.0  13.1  11.0  17.1  11.5
//   term weights, 24 x 768  8.0  10.1   9.8  10.4  11.4  10.5  13.0  10.5  14.8  10.5  19.4  10.5
template <class T, class Epi>
int launch_few8(const Source &h, const uint8_t *mask, int rows, const Weight8 &W, int kp, const Epi &epi, int cus, hipStream_t s) {
    const bool split = (int64_t)W.n < (int64_t)64 * cus;
#define GSV_FEW8(MB)                                                                  \
    return split ? launch_few8<T, MB, kFewWaves, Epi>(h, mask, rows, W, kp, epi, cus, s) \
                 : launch_few8<T, MB, 1, Epi>(h, mask, rows, W, kp, epi, cus, s)
    switch (few_blocks(rows)) {
        case 1: GSV_FEW8(1);
        case 2: GSV_FEW8(2);
        case 4:
            if constexpr (Epi::most_rows > 32) GSV_FEW8(4);
            break;
        default:
            if constexpr (Epi::most_rows > 64) GSV_FEW8(8);
    }
#undef GSV_FEW8
    GS_REQUIRE(false, "%d rows are not few", rows);
}

}  // namespace gsv
