// Rows in 8 bits (gs_int8.h), and linear layers whose weight is kept so:
//   gs_quantize_rows   a matrix's rows as whole numbers and a scale each
//   gs_int8_linear     y = x W^T + b; x is quantised per row within the call, sums are whole numbers
#include "gs_int8.h"

namespace gsv {

// A wave per row.  Bytes bound it (two or four per value in, one out).
template <int HT>
__global__ __launch_bounds__(256) void k_quantize_rows(Source x, int64_t rows, int dimp, int8_t *out, int64_t stride, float *scales, float by) {
    using T = typename HVal<HT>::t;
    const int lane = gs_lane();
    for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < rows; i += (int64_t)gridDim.x * 4) {
        const T *const row[1] = {(const T *)x.p + i * x.s1};
        float scale[1];
        quantize_rows<4, 1>(row, x, dimp, lane, scale, [&](int, int d, uint32_t w) { *reinterpret_cast<uint32_t *>(out + i * stride + d) = w; });
        if (lane == 0) scales[i] = scale[0] * by;
    }
}

int quantize(const Source &x, int type, int64_t rows, int dimp, int8_t *out, int64_t stride, float *scales, float by, hipStream_t s) {
    const dim3 g(gs_blocks(rows, 4, 8192));
#define GSV_QUANTIZE(HT) hipLaunchKernelGGL((k_quantize_rows<HT>), g, dim3(256), 0, s, x, rows, dimp, out, stride, scales, by)
    if (type == GS_H_F32) GSV_QUANTIZE(GS_H_F32);
    else if (type == GS_H_F16) GSV_QUANTIZE(GS_H_F16);
    else GSV_QUANTIZE(GS_H_BF16);
#undef GSV_QUANTIZE
    GS_CHECK_LAUNCH();
    return GS_OK;
}

// A tile's outputs: rows are columns of y (rows of the weight), columns its rows (tokens), so that a lane holds four values on end.
template <class O>
struct EpiLinear {
    const float *w_scales, *x_scales;  // x's times kDown
    const void *bias;
    int bias_type;
    O *out;
    int64_t ld;
    int vec;  // rows of the output are aligned to four values
    static constexpr int sides = 2;
    static constexpr bool row_bias = false;
    __device__ __forceinline__ SideArray side(int a, int r0, int c0, const Shape &s) const {
        return a == 0 ? SideArray{w_scales + r0, s.nr - r0} : SideArray{x_scales + c0, s.nc - c0};
    }
    struct Bias {
        f32x4 b[8];
    };
    template <class TL>
    __device__ __forceinline__ auto before(const Place &at) const {
        Bias h;
        const int q = at.lane >> 4;
#pragma unroll
        for (int i = 0; i < TL::MR; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int v = at.row0 + 16 * i + 4 * q + e;
                h.b[i][e] = bias_at(bias, bias_type, min(v, at.n_r - 1));
            }
        return h;
    }
    template <class TL, class H>
    __device__ __forceinline__ void run(f32x4 (&acc)[TL::MR][TL::MC], const Place &at, const H &held) const {
        const int q = at.lane >> 4;
#pragma unroll
        for (int i = 0; i < TL::MR; i++) {
            const f32x4 sw = at.side4(0, at.r_in + 16 * i + 4 * q);
            const int v = at.row0 + 16 * i + 4 * q;
#pragma unroll
            for (int j = 0; j < TL::MC; j++) {
                const int n = at.col0 + 16 * j + (at.lane & 15);
                const float sx = at.side(1, at.c_in + 16 * j + (at.lane & 15));
                const f32x4 x = __builtin_convertvector(__builtin_bit_cast(i32x4, acc[i][j]), f32x4) * sx * sw;
                f32x4 y;
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = fmaf(x[e], kUp, held.b[i][e]);
                if (n >= at.n_c) continue;
                O *to = out + n * ld + v;
                if (vec && v + 3 < at.n_r) store4(to, y);
                else
                    for (int e = 0; e < 4; e++)
                        if (v + e < at.n_r) to[e] = (O)y[e];
            }
        }
    }
};

// What k_few8 makes of a block's sums: lane l holds rows 16 m + 4 (l >> 4) .. + 3 of column v.
template <class O>
struct EpiFewLinear {
    const void *bias;
    int bias_type;
    O *out;
    template <int MB>
    __device__ __forceinline__ void run(const i32x4 (&acc)[MB], int v, const Weight8 &W, const float *scales, int rows, uint64_t, int q) const {
        if (v >= W.n) return;
        const float by = W.scales[v], b = bias_at(bias, bias_type, v);
#pragma unroll
        for (int m = 0; m < MB; m++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int row = 16 * m + 4 * q + e;
                if (row < rows) out[(int64_t)row * W.n + v] = (O)fmaf((float)acc[m][e] * scales[row] * by, kUp, b);
            }
    }
};

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

Source rows_source(const void *p, int type, int64_t row_stride, int64_t dim_stride, int dim) {
    const bool vec = dim_stride == 1 && row_stride % 4 == 0 && (uintptr_t)p % (type == GS_H_F32 ? 16 : 8) == 0;
    return Source{p, 0, row_stride, dim_stride, 0x7FFFFFFF, dim, vec};
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
    float *scales;
    int dimp;
    bool few;
};
Scratch8 scratch_of(gs_arena &a, const gs_linear8 *l) {
    Scratch8 s{nullptr, nullptr, (int)round_up(l->dim, kPad8), few8_ok(l->rows, (int)round_up(l->dim, kPad8))};
    if (s.few) return s;
    s.scales = a.take<float>(l->rows);
    s.x = a.take<int8_t>((size_t)l->rows * s.dimp);
    return s;
}

template <class O>
int run_product(const gs_linear8 *l, const Scratch8 &s, int cus, hipStream_t st) {
    const Operand w{(const uint16_t *)l->values_d, l->values_stride / 2, 0, s.dimp / 2}, x{(const uint16_t *)s.x, s.dimp / 2, 0, s.dimp / 2};
    const Dims d{l->out, l->rows, s.dimp / 2, nullptr, 0, 0, 0};
    const bool vec = l->out % 4 == 0 && (uintptr_t)l->out_d % (4 * sizeof(O)) == 0;
    const EpiLinear<O> epi{l->scales_d, s.scales, l->bias_d, l->bias_type, (O *)l->out_d, l->out, vec};
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
    return quantize(rows_source(x_d, type, row_stride, dim_stride, dim), type, rows, (int)round_up(dim, kPad8), values_d, values_stride,
                    scales_d, 1.f, gs_stream(stream));
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
    const Source x = rows_source(l->x_d, l->type, l->x_row_stride, l->x_dim_stride, l->dim);
    if (s.few) {
        const Weight8 W{l->values_d, l->values_stride, l->scales_d, l->out};
#define GSV_FEW(HT, O) return launch_few8<typename HVal<HT>::t>(x, nullptr, l->rows, W, s.dimp, EpiFewLinear<O>{l->bias_d, l->bias_type, (O *)l->out_d}, cus, st)
#define GSV_FEW_OUT(HT)                                   \
    if (l->out_type == GS_H_F32) GSV_FEW(HT, float);      \
    if (l->out_type == GS_H_F16) GSV_FEW(HT, _Float16);   \
    GSV_FEW(HT, __bf16)
        if (l->type == GS_H_F32) { GSV_FEW_OUT(GS_H_F32); }
        if (l->type == GS_H_F16) { GSV_FEW_OUT(GS_H_F16); }
        GSV_FEW_OUT(GS_H_BF16);
#undef GSV_FEW_OUT
#undef GSV_FEW
    }
    if (int rc = quantize(x, l->type, l->rows, s.dimp, s.x, s.dimp, s.scales, kDown, st)) return rc;
    if (l->out_type == GS_H_F32) return run_product<float>(l, s, cus, st);
    if (l->out_type == GS_H_F16) return run_product<_Float16>(l, s, cus, st);
    return run_product<__bf16>(l, s, cus, st);
}
