// Values of the types that hidden states, weights and tables come in (GS_H_*), and rows of them.
#pragma once

#include "gs_common.h"

namespace gsv {

typedef float f32x4 __attribute__((ext_vector_type(4)));

__host__ __device__ inline int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

inline bool known(int type) { return type == GS_H_F32 || type == GS_H_F16 || type == GS_H_BF16; }

template <int HT>
struct HVal;
template <>
struct HVal<GS_H_F32> {
    using t = float;
};
template <>
struct HVal<GS_H_F16> {
    using t = _Float16;
};
template <>
struct HVal<GS_H_BF16> {
    using t = __bf16;
};

template <class T>
struct alignas(4 * sizeof(T)) Four {
    T v[4];
};

template <class T>
__device__ __forceinline__ f32x4 load4(const T *p) {
    const Four<T> x = *reinterpret_cast<const Four<T> *>(p);
    return f32x4{(float)x.v[0], (float)x.v[1], (float)x.v[2], (float)x.v[3]};
}
template <class T>
__device__ __forceinline__ void store4(T *p, f32x4 x) {
    *reinterpret_cast<Four<T> *>(p) = Four<T>{{(T)x[0], (T)x[1], (T)x[2], (T)x[3]}};
}

// Up to four values of a row from d on, 0 beyond its end.  `vec`: rows are contiguous and 4-value aligned.
template <class T>
__device__ __forceinline__ f32x4 row4(const T *row, int64_t ds, int d, int dim, bool vec) {
    if (vec && d + 3 < dim) return load4(row + d);
    f32x4 x;
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = d + e < dim ? (float)row[(d + e) * ds] : 0.f;
    return x;
}

struct Source {
    const void *p;
    int64_t s0, s1, sd;  // strides of text, row, value
    int length;          // rows per text
    int dim, vec;
};

template <class T>
__device__ __forceinline__ const T *source_row(const Source &s, int row) {
    return (const T *)s.p + (int64_t)(row / s.length) * s.s0 + (int64_t)(row % s.length) * s.s1;
}

}  // namespace gsv
