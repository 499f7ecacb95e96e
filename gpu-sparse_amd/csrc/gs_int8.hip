// Rows in 8 bits (gs_int8.h), and linear layers whose weight is kept so:
//   gs_quantize_rows   a matrix's rows as whole numbers and a scale each
//   gs_int8_linear     y = x W^T + b; x is quantised per row within the call, sums are whole numbers
#include "gs_int8.h"

namespace gsv {

// A wave per row; workgroups after those write the bias in fp32.  Bytes bound it (two or four per value in, one out): 16384 rows of
// 768 16-bit values 12 us (3.1 TB/s; launch and a row's latency are a third of it).
template <int HT, bool UNIT>
__global__ __launch_bounds__(256) void k_quantize_rows(Source x, int64_t rows, int row_blocks, int dimp, int8_t *out, int64_t stride, float *scales,
                                                       float by, const void *bias, int bias_type, int n, float *bias_o) {
    using T = typename HVal<HT>::t;
    if ((int)blockIdx.x >= row_blocks) {
        const int v = ((int)blockIdx.x - row_blocks) * 256 + (int)threadIdx.x;
        if (v < n) bias_o[v] = bias_at(bias, bias_type, v);
        return;
    }
    const int lane = gs_lane();
    for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < rows; i += (int64_t)row_blocks * 4) {
        const T *row = (const T *)x.p + i * x.s1;
        const float scale = quantize_row<UNIT, 2>(row, row_start<UNIT, 2>(row, x, lane), x, dimp, lane,
                                                  [&](int d, uint2 w) { *reinterpret_cast<uint2 *>(out + i * stride + d) = w; });
        if (lane == 0) scales[i] = scale * by;
    }
}

int quantize(const Source &x, int type, int64_t rows, int dimp, int8_t *out, int64_t stride, float *scales, float by, const void *bias,
             int bias_type, int n, float *bias_o, hipStream_t s) {
    const int row_blocks = (int)gs_blocks(rows, 4, 8192);
    const dim3 g(row_blocks + (n + 255) / 256);
#define GSV_QUANTIZE(HT)                                                                                                                   \
    if (x.sd == 1)                                                                                                                         \
        hipLaunchKernelGGL((k_quantize_rows<HT, true>), g, dim3(256), 0, s, x, rows, row_blocks, dimp, out, stride, scales, by, bias, bias_type, \
                           n, bias_o);                                                                                                     \
    else                                                                                                                                   \
        hipLaunchKernelGGL((k_quantize_rows<HT, false>), g, dim3(256), 0, s, x, rows, row_blocks, dimp, out, stride, scales, by, bias, bias_type, \
                           n, bias_o)
    if (type == GS_H_F32) { GSV_QUANTIZE(GS_H_F32); }
    else if (type == GS_H_F16) { GSV_QUANTIZE(GS_H_F16); }
    else { GSV_QUANTIZE(GS_H_BF16); }
#undef GSV_QUANTIZE
    GS_CHECK_LAUNCH();
    return GS_OK;
}

// Values on end of an output row, which may start anywhere
template <class O, int N>
struct Run {
    typedef O vec __attribute__((ext_vector_type(N), aligned(sizeof(O))));
};

// A tile's outputs: rows are columns of y (rows of the weight), columns its rows (tokens), so that a lane holds four values on
// end.  16-bit ones: lanes of two rows of lanes swap halves, as in store_blocks, so that a lane writes eight.
template <class O>
struct EpiLinear {
    const float *w_scales, *x_scales, *bias;  // x's times kDown
    O *out;
    int64_t ld;
    static constexpr int sides = 3;
    static constexpr bool row_bias = false;
    __device__ __forceinline__ SideArray side(int a, int r0, int c0, const Shape &s) const {
        if (a == 1) return {x_scales + c0, s.nc - c0};
        return {(a == 0 ? w_scales : bias) + r0, s.nr - r0};
    }
    struct None {};
    template <class TL>
    __device__ __forceinline__ None before(const Place &) const {
        return {};
    }
    template <int N>
    __device__ __forceinline__ static void put(O *to, const O (&y)[N], int left) {
        if (left >= N) {
            typename Run<O, N>::vec v;
#pragma unroll
            for (int e = 0; e < N; e++) v[e] = y[e];
            *reinterpret_cast<typename Run<O, N>::vec *>(to) = v;
        } else {
#pragma unroll
            for (int e = 0; e < N; e++)
                if (e < left) to[e] = y[e];
        }
    }
    template <class TL>
    __device__ __forceinline__ void run(f32x4 (&acc)[TL::MR][TL::MC], const Place &at, const None &) const {
        static_assert(TL::MR % 2 == 0, "blocks of rows go in pairs");
        const int q = at.lane >> 4;
#pragma unroll
        for (int j = 0; j < TL::MC; j++) {
            const int n = at.col0 + 16 * j + (at.lane & 15);
            const float sx = at.side(1, at.c_in + 16 * j + (at.lane & 15));
            O *row = out + n * ld;
#pragma unroll
            for (int i = 0; i < TL::MR; i += 2) {
                O y[8];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int in = at.r_in + 16 * (i + h) + 4 * q;
                    const f32x4 x = __builtin_convertvector(__builtin_bit_cast(i32x4, acc[i + h][j]), f32x4) * sx * at.side4(0, in);
                    const f32x4 b = at.side4(2, in);
#pragma unroll
                    for (int e = 0; e < 4; e++) y[4 * h + e] = (O)fmaf(x[e], kUp, b[e]);
                }
                if constexpr (sizeof(O) == 2) {
                    const auto two = [&](int e) {
                        return (uint32_t)__builtin_bit_cast(uint16_t, y[e]) | (uint32_t)__builtin_bit_cast(uint16_t, y[e + 1]) << 16;
                    };
                    const auto u = __builtin_amdgcn_permlane16_swap(two(0), two(4), false, false);
                    const auto v = __builtin_amdgcn_permlane16_swap(two(2), two(6), false, false);
                    const uint32_t w[4] = {u[0], v[0], u[1], v[1]};
#pragma unroll
                    for (int e = 0; e < 8; e++) y[e] = __builtin_bit_cast(O, (uint16_t)(w[e / 2] >> 16 * (e & 1)));
                    const int c = at.row0 + 16 * (i + (q & 1)) + 8 * (q >> 1);
                    if (n < at.n_c) put<8>(row + c, y, at.n_r - c);
                } else {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int c = at.row0 + 16 * (i + h) + 4 * q;
                        const O z[4] = {y[4 * h], y[4 * h + 1], y[4 * h + 2], y[4 * h + 3]};
                        if (n < at.n_c) put<4>(row + c, z, at.n_r - c);
                    }
                }
            }
        }
    }
};

// What k_few8 makes of a block's sums: lane l holds rows 16 m + 4 (l >> 4) .. + 3 of column v.
struct EpiFewLinear {
    const void *bias;
    void *out;
    int bias_type, out_type;
    static constexpr bool joins = false;
    // 24 rows of 768, 30522 columns 10.5 us, in two launches 14; 64 rows 19 and 14: a row's outputs are written 32 bytes at a time
    static constexpr int most_rows = 32;
    __device__ __forceinline__ ColumnScale column(int v, const Weight8 &W) const { return column_scale(v, W, bias, bias_type); }
    __device__ __forceinline__ void block(const i32x4 &sum, int m, int v, const Weight8 &W, const ColumnScale &col, const float *scales, int rows,
                                          int lane, float *) const {
        if (v >= W.n) return;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int row = 16 * m + 4 * (lane >> 4) + e;
            if (row >= rows) continue;
            const float y = fmaf((float)sum[e] * scales[row] * col.by, kUp, col.bias);
            const int64_t to = (int64_t)row * W.n + v;
            if (out_type == GS_H_F32) ((float *)out)[to] = y;
            else if (out_type == GS_H_F16) ((_Float16 *)out)[to] = (_Float16)y;
            else ((__bf16 *)out)[to] = (__bf16)y;
        }
    }
    __device__ __forceinline__ void finish(const float *, int, const Weight8 &, const ColumnScale &, const Kept &, int, int, int) const {}
};

// Tiles: the largest of which there are as many as CUs.  Product alone, us:
//   rows x dim -> out        256      128      64
//   16384 x 1024 -> 4096      76       93     151
//   16384 x 768 -> 768      18.6     18.2      35   (192 tiles of 256: a quarter of the CUs has none)
//   4099 x 777 -> 1001        37       14      14
// The first runs at 1810 TOP/s, of 2404 that a library product of 16384^3 reaches (and of 1280 that it does at this shape); its 134 MB
// of output take 26 us of the 76 at the rate of a copy.
template <class T>
using Small8 = Tile<T, 1, 64, 64, 2, 2, 4, 2, false, false>;
template <class T>
using Mid8 = Tile<T, 1, 128, 128, 2, 2, 2, 2, false, false>;
template <class T>
using Large8 = Tile<T, 1, 256, 256, 2, 4, 2, 2, false, false>;

int check_rows(const char *what, int64_t rows, int dim) {
    GS_REQUIRE(rows >= 0 && rows <= (1 << 28), "%s: %lld rows outside [0, 2^28]", what, (long long)rows);
    GS_REQUIRE(dim >= 1 && dim <= 32768, "%s: dim=%d outside [1, 32768]", what, dim);
    return GS_OK;
}
int check_stride8(const char *what, const void *p, int64_t stride, int dim) {
    GS_REQUIRE(stride % kPad8 == 0 && stride >= round_up(dim, kPad8) && stride < (1 << 20),
               "%s: row stride %lld of 8-bit rows: a multiple of %d, at least dim rounded up to one, below 2^20", what, (long long)stride, kPad8);
    GS_REQUIRE((uintptr_t)p % 16 == 0, "%s: 8-bit rows that are not 16-byte aligned", what);
    return GS_OK;
}

Source rows_source(const void *p, int64_t row_stride, int64_t dim_stride, int dim) {
    return Source{p, 0, row_stride, dim_stride, 0x7FFFFFFF, dim, 0};
}

int check_linear(const gs_linear8 *a) {
    GS_REQUIRE(a, "linear is NULL");
    GS_REQUIRE(known(a->type), "unknown type %d of x", a->type);
    GS_REQUIRE(known(a->out_type), "unknown type %d of the output", a->out_type);
    GS_REQUIRE(known(a->bias_type), "unknown bias type %d", a->bias_type);
    if (int rc = check_rows("int8_linear", a->rows, a->dim)) return rc;
    GS_REQUIRE(a->out >= 1 && a->out <= (1 << 20), "out=%d outside [1, 2^20]", a->out);
    return check_stride8("int8_linear", a->values_d, a->values_stride, a->dim);
}

struct Scratch8 {
    int8_t *x;
    float *scales, *bias;
    int dimp;
    bool few;
};
Scratch8 scratch_of(gs_arena &a, const gs_linear8 *l) {
    Scratch8 s{nullptr, nullptr, nullptr, (int)round_up(l->dim, kPad8), few8_ok<EpiFewLinear>(l->rows, (int)round_up(l->dim, kPad8), l->x_dim_stride)};
    if (s.few) return s;
    s.scales = a.take<float>(l->rows);
    s.bias = a.take<float>(l->out);
    s.x = a.take<int8_t>((size_t)l->rows * s.dimp);
    return s;
}

template <class O>
int run_product(const gs_linear8 *l, const Scratch8 &s, int cus, hipStream_t st) {
    const Operand w{(const uint16_t *)l->values_d, l->values_stride / 2, 0, s.dimp / 2}, x{(const uint16_t *)s.x, s.dimp / 2, 0, s.dimp / 2};
    const Dims d{l->out, l->rows, s.dimp / 2, nullptr, 0, 0, 0};
    const EpiLinear<O> epi{l->scales_d, s.scales, s.bias, (O *)l->out_d, l->out};
    const auto tiles = [&](int e) { return (int64_t)((l->out + e - 1) / e) * ((l->rows + e - 1) / e); };
    if (tiles(256) >= cus) return launch_product<Large8<I8>>(w, x, d, epi, cus, st);
    if (tiles(128) >= cus) return launch_product<Mid8<I8>>(w, x, d, epi, cus, st);
    return launch_product<Small8<I8>>(w, x, d, epi, cus, st);
}

}  // namespace gsv

using namespace gsv;

extern "C" int gs_quantize_rows(const void *x_d, int32_t type, int64_t rows, int32_t dim, int64_t row_stride, int64_t dim_stride,
                                int8_t *values_d, int64_t values_stride, float *scales_d, void *stream) {
    GS_REQUIRE(known(type), "unknown type %d", type);
    if (int rc = check_rows("quantize_rows", rows, dim)) return rc;
    if (int rc = check_stride8("quantize_rows", values_d, values_stride, dim)) return rc;
    if (rows == 0) return GS_OK;
    GS_REQUIRE(x_d && values_d && scales_d, "NULL rows, values or scales");
    return quantize(rows_source(x_d, row_stride, dim_stride, dim), type, rows, (int)round_up(dim, kPad8), values_d, values_stride,
                    scales_d, 1.f, nullptr, GS_H_F32, 0, nullptr, gs_stream(stream));
}

extern "C" int gs_int8_linear_workspace(const gs_linear8 *l, size_t *bytes) {
    if (int rc = check_linear(l)) return rc;
    GS_REQUIRE(bytes, "NULL size pointer");
    gs_arena a{nullptr, 0, 0};
    scratch_of(a, l);
    *bytes = a.used;
    return GS_OK;
}

extern "C" int gs_int8_linear(const gs_linear8 *l, void *workspace_d, size_t workspace_bytes, void *stream) {
    if (int rc = check_linear(l)) return rc;
    gs_arena a{(char *)workspace_d, 0, workspace_bytes};
    const Scratch8 s = scratch_of(a, l);
    if (!a.ok()) {
        gs_set_error("int8_linear workspace too small: need %zu bytes, got %zu", a.used, workspace_bytes);
        return GS_ENOSPC;
    }
    if (l->rows == 0) return GS_OK;
    GS_REQUIRE(l->x_d && l->values_d && l->scales_d && l->out_d && (workspace_d || a.used == 0), "NULL x, weight, output or workspace");
    int cus = 0;
    if (int rc = cu_count(&cus)) return rc;
    const hipStream_t st = gs_stream(stream);
    const Source x = rows_source(l->x_d, l->x_row_stride, l->x_dim_stride, l->dim);
    if (s.few) {
        const Weight8 W{l->values_d, l->values_stride, l->scales_d, l->out};
        const EpiFewLinear epi{l->bias_d, l->out_d, l->bias_type, l->out_type};
        if (l->type == GS_H_F32) return launch_few8<float>(x, nullptr, l->rows, W, s.dimp, epi, cus, st);
        if (l->type == GS_H_F16) return launch_few8<_Float16>(x, nullptr, l->rows, W, s.dimp, epi, cus, st);
        return launch_few8<__bf16>(x, nullptr, l->rows, W, s.dimp, epi, cus, st);
    }
    if (int rc = quantize(x, l->type, l->rows, s.dimp, s.x, s.dimp, s.scales, kDown, l->bias_d, l->bias_type, l->out, s.bias, st)) return rc;
    if (l->out_type == GS_H_F32) return run_product<float>(l, s, cus, st);
    if (l->out_type == GS_H_F16) return run_product<_Float16>(l, s, cus, st);
    return run_product<__bf16>(l, s, cus, st);
}
