// The vocabulary head of a learned sparse encoder: l = h W^T + b over the vocabulary, with
//   gs_term_weights   w[b][v] = log(1 + relu(max over a text's kept tokens of l)), and its gradient
//   gs_vocab_loss     softmax cross entropy, or distillation from a teacher's top logits, and their gradients
// The logits are made tile by tile (gs_vocab_gemm.h) and consumed in registers.  The losses' gradients make them
// again, a piece of the vocabulary at a time, as gradients in 16 bits that two more products read.
#include <math.h>

#include "gs_vocab_gemm.h"

namespace gsv {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr int kRowPad = 256;           // rows of the vocabulary are padded to this (bias -inf beyond the last)
constexpr int kMaxTop = 1024;          // teacher logits per row
constexpr size_t kPieceBytes = 512u << 20;  // logit gradients held at a time

__host__ __device__ inline int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

// ---------------------------------------------------------------- values

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

template <class T>
__device__ __forceinline__ uint16_t bits16(float x) {
    return __builtin_bit_cast(uint16_t, (T)x);
}

// x as bf16 planes, each the nearest to what is left.  A value that is not finite is its first plane alone.
__device__ __forceinline__ void split3(float x, uint16_t (&p)[3]) {
    const __bf16 a = (__bf16)x;
    const float r = x - (float)a;
    const __bf16 b = (__bf16)r;
    const __bf16 c = (__bf16)(r - (float)b);
    const bool fin = fabsf(x) < 3.3e38f;
    p[0] = __builtin_bit_cast(uint16_t, a);
    p[1] = fin ? __builtin_bit_cast(uint16_t, b) : 0;
    p[2] = fin ? __builtin_bit_cast(uint16_t, c) : 0;
}

template <class T, int NP>
__device__ __forceinline__ void store_planes4(uint16_t *row, int64_t plane, int d, f32x4 x) {
    if constexpr (NP == 1) {
        *reinterpret_cast<Four<uint16_t> *>(row + d) =
            Four<uint16_t>{{bits16<T>(x[0]), bits16<T>(x[1]), bits16<T>(x[2]), bits16<T>(x[3])}};
    } else {
        Four<uint16_t> o[3];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            uint16_t p[3];
            split3(x[e], p);
            o[0].v[e] = p[0], o[1].v[e] = p[1], o[2].v[e] = p[2];
        }
#pragma unroll
        for (int i = 0; i < 3; i++) *reinterpret_cast<Four<uint16_t> *>(row + i * plane + d) = o[i];
    }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, GS_WAVE);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, GS_WAVE));
    return v;
}
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}
// over the 16 lanes of a row of lanes
__device__ __forceinline__ float sum16(float v) { return dpp_add<0x121>(dpp_add<0x122>(dpp_add<0x124>(dpp_add<0x128>(v)))); }

// ---------------------------------------------------------------- kept rows

// rows[i]: the i-th row with keep[row] != 0, ascending (keep NULL: all); inv[row]: its place or -1; *n: how many.
// For texts of `length` rows, seg[i] is the row's text.  One workgroup, 16 rows per thread and turn.
__global__ __launch_bounds__(1024) void k_kept_rows(const uint8_t *keep, int total, int length, int *rows, int *inv,
                                                    int *seg, int *n) {
    __shared__ int part[16];
    __shared__ int base_s;
    const int tid = threadIdx.x, lane = gs_lane(), wave = tid >> 6;
    int base = 0;
    const bool vec = keep && (reinterpret_cast<uintptr_t>(keep) & 15) == 0;
    for (int64_t at = 0; at < total; at += 16384) {
        const int64_t r0 = at + tid * 16;
        uint32_t m = 0;
        if (r0 < total) {
            if (!keep) m = 0xFFFF;
            else if (vec && r0 + 16 <= total) {
                const uint4 w = *reinterpret_cast<const uint4 *>(keep + r0);
                const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int e = 0; e < 16; e++) m |= (((ws[e >> 2] >> (8 * (e & 3))) & 255u) ? 1u : 0u) << e;
            } else {
                for (int e = 0; e < 16 && r0 + e < total; e++) m |= (keep[r0 + e] ? 1u : 0u) << e;
            }
            if (r0 + 16 > total) m &= (1u << (total - r0)) - 1u;
        }
        const uint32_t c = __popc(m);
        const uint32_t inc = gs_wave_incl_scan(c);
        if (lane == 63) part[wave] = (int)inc;
        __syncthreads();
        int before = base;
        for (int w = 0; w < wave; w++) before += part[w];
        if (tid == 1023) base_s = before + (int)inc;
        int o = before + (int)(inc - c);
        for (int e = 0; e < 16 && r0 + e < total; e++) {
            const bool k = (m >> e) & 1;
            const int row = (int)(r0 + e);
            if (inv) inv[row] = k ? o : -1;
            if (k) {
                rows[o] = row;
                if (seg) seg[o] = row / length;
                o++;
            }
        }
        __syncthreads();
        base = base_s;
        __syncthreads();
    }
    if (tid == 0) *n = base;
}

// ---------------------------------------------------------------- packing

struct Source {
    const void *p;
    int64_t s0, s1, sd;  // strides of text, row, value
    int length;          // rows per text
    int dim, vec;
};

// Rows of a strided matrix as contiguous 16-bit ones (fp32: three planes), zero to a multiple of kStep values.
template <int HT, int NP>
__global__ __launch_bounds__(256) void k_pack(Source s, const int *rows, const int *n_d, int n, int dimp, uint16_t *out) {
    using T = typename HVal<HT>::t;
    using S = std::conditional_t<HT == GS_H_F16, _Float16, __bf16>;
    if (n_d) n = min(n, *n_d);
    const int lane = gs_lane();
    for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < n; i += (int64_t)gridDim.x * 4) {
        const int row = rows ? rows[i] : (int)i;
        const T *src = (const T *)s.p + (int64_t)(row / s.length) * s.s0 + (int64_t)(row % s.length) * s.s1;
        uint16_t *dst = out + i * (int64_t)NP * dimp;
        for (int d = lane * 4; d < dimp; d += 256) store_planes4<S, NP>(dst, dimp, d, row4(src, s.sd, d, s.dim, s.vec));
    }
}

// The bias in fp32 (0 without one), -inf for the rows that pad the vocabulary: they drop out of every softmax.
__global__ void k_bias(const void *bias, int type, int vocab, int padded, float *out) {
    const int v = blockIdx.x * blockDim.x + threadIdx.x;
    if (v >= padded) return;
    float x = 0.f;
    if (v >= vocab) x = -INFINITY;
    else if (bias)
        x = type == GS_H_F32 ? ((const float *)bias)[v]
                             : type == GS_H_F16 ? (float)((const _Float16 *)bias)[v] : (float)((const __bf16 *)bias)[v];
    out[v] = x;
}

// ---------------------------------------------------------------- targets

// One target per row: its id, and whether the row counts (an id outside the vocabulary does not, as in a search).
__global__ void k_targets(const int64_t *targets, int64_t ignore, int rows, int vocab, int *ids, uint8_t *keep) {
    const int r = blockIdx.x * blockDim.x + threadIdx.x;
    if (r >= rows) return;
    const int64_t t = targets[r];
    const bool ok = t >= 0 && t < vocab && t != ignore;
    ids[r] = ok ? (int)t : -1;
    keep[r] = ok;
}

// A teacher's row: q = softmax(logits / tau) over its ids inside the vocabulary, sorted by id (equal ids stay apart,
// in their order), ids beyond them INT_MAX; sum of q log q.  One workgroup per row; LDS holds the row.
__global__ __launch_bounds__(256) void k_teacher(const int64_t *ids, const void *logits, int type, int top, int vocab,
                                                 float inv_tau, int *ids_o, float *q_o, float *ent_o, uint8_t *keep) {
    __shared__ int sid[kMaxTop];
    __shared__ float sz[kMaxTop];
    __shared__ float red[8];
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x, wave = tid >> 6, nw = blockDim.x >> 6;
    auto block = [&](float v, bool sum) {
        v = sum ? wave_sum(v) : wave_max(v);
        __syncthreads();
        if (gs_lane() == 0) red[wave] = v;
        __syncthreads();
        float o = red[0];
        for (int w = 1; w < nw; w++) o = sum ? o + red[w] : fmaxf(o, red[w]);
        return o;
    };
    float most = -INFINITY;
    int any = 0;
    for (int k = tid; k < top; k += blockDim.x) {
        const int64_t id = ids[r * top + k];
        const bool ok = id >= 0 && id < vocab;
        const int64_t at = r * top + k;
        float z = type == GS_H_F32 ? ((const float *)logits)[at]
                                   : type == GS_H_F16 ? (float)((const _Float16 *)logits)[at] : (float)((const __bf16 *)logits)[at];
        z *= inv_tau;
        sid[k] = ok ? (int)id : 0x7FFFFFFF;
        sz[k] = z;
        any |= ok;
        if (ok) most = fmaxf(most, z);
    }
    most = block(most, false);
    any = __syncthreads_or(any);
    float s = 0.f;
    for (int k = tid; k < top; k += blockDim.x) {
        const float e = sid[k] == 0x7FFFFFFF ? 0.f : expf(sz[k] - most);
        sz[k] = e;
        s += e;
    }
    s = block(s, true);
    const float inv = 1.f / s;
    float ent = 0.f;
    for (int k = tid; k < top; k += blockDim.x) {
        const int id = sid[k];
        const float q = id == 0x7FFFFFFF ? 0.f : sz[k] * inv;
        if (q != 0.f) ent += q * logf(q);
        int at = 0;
        for (int j = 0; j < top; j++) at += sid[j] < id || (sid[j] == id && j < k);
        ids_o[r * top + at] = id;
        q_o[r * top + at] = q;
    }
    ent = block(ent, true);
    if (tid == 0) {
        ent_o[r] = ent;
        keep[r] = any != 0;
    }
}

// first[t][i]: where row rows[i]'s entries with ids >= t * width begin (K > 1 only)
__global__ void k_entry_starts(const int *ids, int top, const int *rows, const int *n_d, int tiles, int width, int64_t ld,
                               uint16_t *first) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= *n_d) return;
    const int *row = ids + (int64_t)rows[i] * top;
    int k = 0;
    for (int t = 0; t <= tiles; t++) {
        const int64_t v = (int64_t)t * width;
        while (k < top && row[k] < v) k++;
        first[t * ld + i] = (uint16_t)k;
    }
}

// sum_k q_k l[id_k] of each kept row, from the unpacked values in fp32.  One wave per row, ids in turn.
template <int HT>
__global__ __launch_bounds__(256) void k_target_logits(Source h, const void *weight, int64_t wr, int64_t wd, int wvec,
                                                       const float *bias, const int *ids, const float *q, int top,
                                                       const int *rows, const int *n_d, float *out) {
    using T = typename HVal<HT>::t;
    const int n = *n_d, lane = gs_lane();
    for (int i = blockIdx.x * 4 + (threadIdx.x >> 6); i < n; i += gridDim.x * 4) {
        const int row = rows[i];
        const T *src = (const T *)h.p + (int64_t)(row / h.length) * h.s0 + (int64_t)(row % h.length) * h.s1;
        float sum = 0.f;
        for (int k0 = 0; k0 < top; k0 += 4) {
            int id[4];
            float qk[4], a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int k = k0 + e;
                id[e] = k < top ? ids[(int64_t)row * top + k] : 0x7FFFFFFF;
                qk[e] = id[e] == 0x7FFFFFFF || id[e] < 0 ? 0.f : q ? q[(int64_t)row * top + k] : 1.f;
                if (qk[e] == 0.f) id[e] = -1;
            }
            if ((id[0] & id[1] & id[2] & id[3]) < 0 && id[0] < 0 && id[1] < 0 && id[2] < 0 && id[3] < 0) continue;
            for (int d = lane * 4; d < h.dim; d += 256) {
                const f32x4 x = row4(src, h.sd, d, h.dim, h.vec);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (id[e] < 0) continue;
                    const f32x4 y = row4((const T *)weight + id[e] * wr, wd, d, h.dim, wvec);
                    a[e] = fmaf(x[0], y[0], fmaf(x[1], y[1], fmaf(x[2], y[2], fmaf(x[3], y[3], a[e]))));
                }
            }
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (id[e] >= 0) sum += qk[e] * (wave_sum(a[e]) + bias[id[e]]);
        }
        if (lane == 0) out[i] = sum;
    }
}

// ---------------------------------------------------------------- epilogues

// Softmax sums of a tile: per token the largest scaled logit and the sum of 2^(scaled logit - it), over each wave's
// terms.  part[block of terms][token].
struct EpiSums {
    const float *bias;
    float scale;  // log2(e) / temperature
    float2 *part;
    int64_t ld;
    template <class TL>
    __device__ __forceinline__ void run(f32x4 (&acc)[TL::MR][TL::MC], const Place &at) const {
        const int q = at.lane >> 4;
#pragma unroll
        for (int i = 0; i < TL::MR; i++) {
            const f32x4 b = *reinterpret_cast<const f32x4 *>(bias + at.row0 + 16 * i + 4 * q);
#pragma unroll
            for (int j = 0; j < TL::MC; j++) acc[i][j] += b;
        }
        const int64_t block = at.row0 / (TL::MR * 16);
#pragma unroll
        for (int j = 0; j < TL::MC; j++) {
            float m = -INFINITY;
#pragma unroll
            for (int i = 0; i < TL::MR; i++)
                m = fmaxf(m, fmaxf(fmaxf(acc[i][j][0], acc[i][j][1]), fmaxf(acc[i][j][2], acc[i][j][3])));
            float mc = m * scale, s = 0.f;
            const float sub = m == -INFINITY ? 0.f : mc;
#pragma unroll
            for (int i = 0; i < TL::MR; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) s += __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], scale, -sub));
#pragma unroll
            for (int d = 16; d <= 32; d <<= 1) {
                const float mo = __shfl_xor(mc, d, GS_WAVE), so = __shfl_xor(s, d, GS_WAVE);
                const float mn = fmaxf(mc, mo), by = mn == -INFINITY ? 0.f : mn;
                s = s * __builtin_amdgcn_exp2f(mc - by) + so * __builtin_amdgcn_exp2f(mo - by);
                mc = mn;
            }
            const int n = at.col0 + 16 * j + (at.lane & 15);
            if (q == 0 && n < at.n_c) part[block * ld + n] = make_float2(mc, s);
        }
    }
};

// Gradients of a tile's logits: (softmax - target shares) times the row's factor, rounded to 16 bits once (three
// planes for fp32), token-major, and their sums over each wave's tokens for the bias.
template <class S>
struct EpiLogitGrad {
    const float *bias;
    float scale;
    const float *lse2;     // log2 of the softmax sum, per kept row
    const float *factor;   // per kept row
    const int *rows;       // kept row -> source row
    const int *ids;        // [source row][top], ascending
    const float *share;    // NULL: 1
    const uint16_t *first; // [vocabulary / kRowPad][kept row] (top > 1)
    int64_t first_ld;
    int top;
    int v0;                // first term of this piece
    uint16_t *out;
    int64_t ld, plane;
    float *col_sums;       // NULL: not wanted; [wave's block of tokens][padded vocabulary]
    int64_t sums_ld;
    template <class TL>
    __device__ __forceinline__ void run(f32x4 (&acc)[TL::MR][TL::MC], const Place &at) const {
        const int q = at.lane >> 4;
        f32x4 sums[TL::MR];
#pragma unroll
        for (int i = 0; i < TL::MR; i++) {
            sums[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            const f32x4 b = *reinterpret_cast<const f32x4 *>(bias + v0 + at.row0 + 16 * i + 4 * q);
#pragma unroll
            for (int j = 0; j < TL::MC; j++) acc[i][j] += b;
        }
        const int wv = v0 + at.row0;  // the wave's first term
#pragma unroll
        for (int j = 0; j < TL::MC; j++) {
            const int n = at.col0 + 16 * j + (at.lane & 15);
            const bool on = n < at.n_c;
            const float l = on ? lse2[n] : 0.f, f = on ? factor[n] : 0.f;
#pragma unroll
            for (int i = 0; i < TL::MR; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[i][j][e] = __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], scale, -l));
            // target shares: the lane that holds the entry's term takes them off
            int64_t base = 0;
            int k = 0, end = 0;
            if (on) {
                base = (int64_t)rows[n] * top;
                end = top;
                if (top > 1) {
                    const int t = wv / kRowPad;
                    k = first[t * first_ld + n];
                    end = first[(t + 1) * first_ld + n];
                }
            }
            int id = k < end ? ids[base + k] : 0x7FFFFFFF;
            while (__any(k < end)) {
                const int lv = id - wv;
                if (__any(k < end && lv >= 0 && lv < TL::MR * 16)) {
                    const float s = k < end ? (share ? share[base + k] : 1.f) : 0.f;
                    const int mine = k < end && lv >= 0 && ((lv >> 2) & 3) == q ? (lv >> 4) * 4 + (lv & 3) : -1;
#pragma unroll
                    for (int i = 0; i < TL::MR; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[i][j][e] -= mine == i * 4 + e ? s : 0.f;
                }
                k++;
                id = k < end ? ids[base + k] : 0x7FFFFFFF;
            }
#pragma unroll
            for (int i = 0; i < TL::MR; i++) {
                acc[i][j] *= f;
                sums[i] += on ? acc[i][j] : f32x4{0.f, 0.f, 0.f, 0.f};
                if (on) store_planes4<S, TL::planes>(out + n * ld, plane, at.row0 + 16 * i + 4 * q, acc[i][j]);
            }
        }
        if (col_sums) {
            float *to = col_sums + (int64_t)(at.col0 / (TL::MC * 16)) * sums_ld + wv;
#pragma unroll
            for (int i = 0; i < TL::MR; i++) {
                f32x4 s;
#pragma unroll
                for (int e = 0; e < 4; e++) s[e] = sum16(sums[i][e]);
                if ((at.lane & 15) == 0) *reinterpret_cast<f32x4 *>(to + 16 * i + 4 * q) = s;
            }
        }
    }
};

// dW: rows are dim, columns terms; out[term][dim] times *scale
template <class O>
struct EpiWeightGrad {
    O *out;
    const float *scale;
    int dim, vec;
    template <class TL>
    __device__ __forceinline__ void run(f32x4 (&acc)[TL::MR][TL::MC], const Place &at) const {
        const float s = *scale;
        const int q = at.lane >> 4;
#pragma unroll
        for (int j = 0; j < TL::MC; j++) {
            const int v = at.col0 + 16 * j + (at.lane & 15);
            if (v >= at.n_c) continue;
            O *to = out + (int64_t)v * dim;
#pragma unroll
            for (int i = 0; i < TL::MR; i++) {
                const int d = at.row0 + 16 * i + 4 * q;
                const f32x4 x = acc[i][j] * s;
                if (vec && d + 3 < dim) store4(to + d, x);
                else
                    for (int e = 0; e < 4; e++)
                        if (d + e < dim) to[d + e] = (O)x[e];
            }
        }
    }
};

// dH in parts: rows are dim, columns kept rows; part[split][kept row][dim], added to what earlier pieces left
struct EpiHiddenPart {
    float *part;
    int dimp, add;
    template <class TL>
    __device__ __forceinline__ void run(f32x4 (&acc)[TL::MR][TL::MC], const Place &at) const {
        const int q = at.lane >> 4;
#pragma unroll
        for (int j = 0; j < TL::MC; j++) {
            const int n = at.col0 + 16 * j + (at.lane & 15);
            if (n >= at.n_c) continue;
            float *to = part + ((int64_t)at.split * at.n_c + n) * dimp;
#pragma unroll
            for (int i = 0; i < TL::MR; i++) {
                const int d = at.row0 + 16 * i + 4 * q;
                if (d >= dimp) continue;
                f32x4 x = acc[i][j];
                if (add) x += *reinterpret_cast<const f32x4 *>(to + d);
                *reinterpret_cast<f32x4 *>(to + d) = x;
            }
        }
    }
};

// Largest logit of each text and term: rows are kept tokens (ascending by text), columns terms.  best[text][term]
// takes the maximum of the positive ones' bits; with tokens, of (bits, ~kept row), so that the lowest token wins a
// tie.  Maxima do not depend on the order of the atomics.
template <bool TOK>
struct EpiTextMax {
    const float *bias;
    const int *seg;   // text of each kept row, padded with -1 to a whole tile
    void *best;
    int vocab;
    template <class TL>
    __device__ __forceinline__ void run(f32x4 (&acc)[TL::MR][TL::MC], const Place &at) const {
        static_assert(TL::MC <= 4, "a lane group flushes one column block");
        const int q = at.lane >> 4;
        float b[TL::MC];
#pragma unroll
        for (int j = 0; j < TL::MC; j++) b[j] = bias[at.col0 + 16 * j + (at.lane & 15)];
        int cur = -1;
        float top[TL::MC];
        int tok[TL::MC];
        auto flush = [&]() {
            if (cur < 0) return;
            float mine = 0.f;
            int row = 0;
#pragma unroll
            for (int j = 0; j < TL::MC; j++) {
                float x = top[j];
                int r = tok[j];
#pragma unroll
                for (int d = 16; d <= 32; d <<= 1) {
                    const float xo = __shfl_xor(x, d, GS_WAVE);
                    if (TOK) {
                        const int ro = __shfl_xor(r, d, GS_WAVE);
                        const bool take = __float_as_int(xo) > __float_as_int(x) || (__float_as_int(xo) == __float_as_int(x) && ro < r);
                        x = take ? xo : x;
                        r = take ? ro : r;
                    } else {
                        x = __int_as_float(max(__float_as_int(x), __float_as_int(xo)));
                    }
                }
                if (j == q) mine = x, row = r;
            }
            const int v = at.col0 + 16 * q + (at.lane & 15);
            if (q < TL::MC && v < vocab && __float_as_int(mine) > 0) {
                const int64_t o = (int64_t)cur * vocab + v;
                if (TOK) {
                    const unsigned long long key = (unsigned long long)__float_as_uint(mine) << 32 | (0xFFFFFFFFu - (uint32_t)row);
                    atomicMax((unsigned long long *)best + o, key);
                } else {
                    atomicMax((uint32_t *)best + o, __float_as_uint(mine));
                }
            }
        };
#pragma unroll
        for (int i = 0; i < TL::MR; i++) {
            const int row = at.row0 + 16 * i + 4 * q;
            const int4 s = *reinterpret_cast<const int4 *>(seg + row);
            const int lo = __builtin_amdgcn_readlane(s.x, 0);
            // as integers, positive values and NaN order as wanted and negative ones lie below the start, 0
            const int sv[4] = {s.x, s.y, s.z, s.w};
            int now = lo;
            while (now >= 0) {
                if (now != cur) {
                    flush();
                    cur = now;
#pragma unroll
                    for (int j = 0; j < TL::MC; j++) top[j] = 0.f, tok[j] = 0x7FFFFFFF;
                }
#pragma unroll
                for (int j = 0; j < TL::MC; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float raw = acc[i][j][e] + b[j];
                        const float x = sv[e] == now ? (raw != raw ? __int_as_float(0x7FC00000) : raw) : 0.f;
                        if (TOK) {
                            const bool take = __float_as_int(x) > __float_as_int(top[j]);
                            top[j] = take ? x : top[j];
                            tok[j] = take ? row + e : tok[j];
                        } else {
                            top[j] = __int_as_float(max(__float_as_int(top[j]), __float_as_int(x)));
                        }
                    }
                // the next text in this block, if any
                int next = 0x7FFFFFFF;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (sv[e] > now) next = min(next, sv[e]);
                next = min(next, __shfl_xor(next, 16, GS_WAVE));
                next = min(next, __shfl_xor(next, 32, GS_WAVE));
                next = gs_uniform(next);
                now = next == 0x7FFFFFFF ? -1 : next;
            }
        }
        flush();
    }
};

// ---------------------------------------------------------------- losses' small kernels

// log2 of each kept row's softmax sum, and its loss.  Sixteen rows per 256 threads.
__global__ __launch_bounds__(256) void k_row_loss(const float2 *part, int64_t ld, int blocks, const int *rows, const int *n_d,
                                                  const float *target, const float *ent, float tau, float *lse2_o,
                                                  float *loss_o, float *loss_rows) {
    __shared__ float sm[16][17], ss[16][17];
    const int n = *n_d, x = threadIdx.x & 15, y = threadIdx.x >> 4;
    for (int64_t i0 = (int64_t)blockIdx.x * 16; i0 < n; i0 += (int64_t)gridDim.x * 16) {
        const int64_t i = i0 + x;
        float m = -INFINITY, s = 0.f;
        if (i < n)
            for (int b = y; b < blocks; b += 16) {
                const float2 p = part[b * ld + i];
                const float mn = fmaxf(m, p.x), by = mn == -INFINITY ? 0.f : mn;
                s = s * __builtin_amdgcn_exp2f(m - by) + p.y * __builtin_amdgcn_exp2f(p.x - by);
                m = mn;
            }
        sm[y][x] = m;
        ss[y][x] = s;
        __syncthreads();
        if (y == 0 && i < n) {
            for (int b = 1; b < 16; b++) {
                const float mn = fmaxf(m, sm[b][x]), by = mn == -INFINITY ? 0.f : mn;
                s = s * __builtin_amdgcn_exp2f(m - by) + ss[b][x] * __builtin_amdgcn_exp2f(sm[b][x] - by);
                m = mn;
            }
            const float l2 = m + log2f(s);
            const int row = rows[i];
            const float loss = tau * tau * ((ent ? ent[row] : 0.f) + (l2 * kLn2 - target[i] / tau));
            lse2_o[i] = l2;
            loss_o[i] = loss;
            if (loss_rows) loss_rows[row] = loss;
        }
        __syncthreads();
    }
}

__global__ void k_fill(float *p, int64_t n, float v) {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) p[i] = v;
}

// Sum (or mean) of the kept rows' losses, in an order of its own; 0 where no row is kept.
__global__ __launch_bounds__(1024) void k_loss_sum(const float *loss, const int *n_d, int mean, float *out) {
    __shared__ double part[16];
    const int n = *n_d;
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 1024) s += (double)loss[i];
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d, GS_WAVE);
    if (gs_lane() == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; w++) s += part[w];
        *out = n == 0 ? 0.f : (float)(mean ? s / n : s);
    }
}

// What a kept row's logit gradient is multiplied with before it is rounded to 16 bits, and what the sums over such
// gradients are: scale[0].  With one upstream value for all rows that value is kept out of the rounding, so that the
// largest parts, p - 1 at a target, are rounded next to 1, where they almost lie.  Values of their own (one per row)
// go into the gradients.  fp16's range asks for a power of two as well: |p - share| <= 1, so the gradients' largest
// magnitude is put at 2^11 to 2^12.
__global__ __launch_bounds__(1024) void k_row_factor(const float *grad, int per_row, const int *rows, const int *n_d, int mean,
                                                     float tau, int f16, float *factor, float *scale) {
    __shared__ float part[16];
    const int n = *n_d;
    if (!per_row) {
        const float up = f16 ? 2048.f : 1.f;
        for (int i = threadIdx.x; i < n; i += 1024) factor[i] = up;
        if (threadIdx.x == 0) scale[0] = grad[0] * (mean ? tau / (float)max(n, 1) : tau) / up;
        return;
    }
    float most = 0.f;
    for (int i = threadIdx.x; i < n; i += 1024) {
        const float f = grad[rows[i]] * tau;
        factor[i] = f;
        most = fmaxf(most, fabsf(f));
    }
    float up = 1.f;
    if (f16) {
        most = wave_max(most);
        if (gs_lane() == 0) part[threadIdx.x >> 6] = most;
        __syncthreads();
        most = part[0];
        for (int w = 1; w < 16; w++) most = fmaxf(most, part[w]);
        if (most > 0.f && most < 3e38f) {
            up = ldexpf(1.f, max(-120, min(120, 11 - ilogbf(most))));
            for (int i = threadIdx.x; i < n; i += 1024) factor[i] *= up;
        }
    }
    if (threadIdx.x == 0) scale[0] = 1.f / up;
}

// dH of every source row from its parts (0 for rows that are not kept)
template <class O>
__global__ __launch_bounds__(256) void k_hidden_grad(const float *part, const int *inv, const int *n_d, int total, int dim,
                                                     int dimp, int tr, int bc, int slots, int most,
                                                     const float *scale, O *out) {
    const int n = *n_d, lane = gs_lane();
    const int split = parts_of(n, tr, bc, slots, most);
    const float s = *scale;
    const bool vec = (dim & 3) == 0;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < total; r += (int64_t)gridDim.x * 4) {
        const int i = inv[r];
        for (int d = lane * 4; d < dim; d += 256) {
            f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
            if (i >= 0)
                for (int p = 0; p < split; p++) x += *reinterpret_cast<const f32x4 *>(part + ((int64_t)p * n + i) * dimp + d);
            x *= s;
            O *to = out + r * dim + d;
            if (vec) store4(to, x);
            else
                for (int e = 0; e < 4; e++)
                    if (d + e < dim) to[e] = (O)x[e];
        }
    }
}

// db: the tiles' column sums added up in order
template <class O>
__global__ __launch_bounds__(256) void k_bias_grad(const float *sums, int64_t ld, const int *n_d, int bc, int per_tile, int vocab,
                                                   const float *scale, O *out) {
    const int v = blockIdx.x * 256 + threadIdx.x;
    if (v >= vocab) return;
    const int blocks = (*n_d + bc - 1) / bc * per_tile;
    float s = 0.f;
    for (int b = 0; b < blocks; b++) s += sums[b * ld + v];
    out[v] = (O)(s * *scale);
}

// ---------------------------------------------------------------- term weights' small kernels

template <bool TOK>
__global__ void k_term_weights(const void *best, int64_t n, int vocab, const int *rows, int length, float *weights,
                               int *tokens) {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        if (TOK) {
            const unsigned long long k = ((const unsigned long long *)best)[i];
            weights[i] = log1pf(__uint_as_float((uint32_t)(k >> 32)));
            tokens[i] = k ? rows[0xFFFFFFFFu - (uint32_t)k] % length : -1;
        } else {
            weights[i] = log1pf(__uint_as_float(((const uint32_t *)best)[i]));
        }
    }
}

// Entries of one text sorted by token, terms ascending within a token: entry_v / entry_g[text * vocab ...], and the
// first entry of each token (first[text][length + 1]).  One workgroup per text.  Each wave owns a run of terms, so a
// count per (wave, token) places every entry without an atomic that decides an order; tokens go in passes of kTok.
constexpr int kTok = 512, kSortWaves = 16;
__global__ __launch_bounds__(1024) void k_sort_entries(const float *grad, const float *weights, const int *tokens, int vocab,
                                                       int length, float *entry_g, int *entry_v, int *first) {
    __shared__ int count[kSortWaves][kTok];
    __shared__ int start[kTok];
    __shared__ int wsum[16];
    const int64_t b = blockIdx.x;
    const int tid = threadIdx.x, lane = gs_lane(), wave = tid >> 6;
    const float *g = grad + b * vocab, *w = weights + b * vocab;
    const int *tk = tokens + b * vocab;
    const int run = (int)round_up((vocab + kSortWaves - 1) / kSortWaves, 64);
    const int lo = min(vocab, wave * run), hi = min(vocab, lo + run);
    int base = 0;
    for (int t0 = 0; t0 < length; t0 += kTok) {
        for (int t = lane; t < kTok; t += 64) count[wave][t] = 0;
        gs_wave_sync();
        auto walk = [&](bool place) {
            for (int v0 = lo; v0 < hi; v0 += 64) {
                const int v = v0 + lane;
                const int t = v < hi ? tk[v] - t0 : -1;
                const bool on = t >= 0 && t < kTok && t0 + t < length;
                uint64_t left = __ballot(on);
                int rank = 0, all = 0;
                while (left) {  // one turn per distinct token among the lanes
                    const int lead = __ffsll((unsigned long long)left) - 1;
                    const int tl = __builtin_amdgcn_readlane(t, lead);
                    const uint64_t same = __ballot(on && t == tl);
                    if (on && t == tl) {
                        rank = __popcll(same & gs_lanemask_lt());
                        all = __popcll(same);
                    }
                    left &= ~same;
                }
                if (on) {
                    const int had = count[wave][t];
                    if (place) {
                        const int64_t at = b * vocab + start[t] + had + rank;
                        entry_v[at] = v;
                        entry_g[at] = g[v] * expf(-w[v]);  // d log(1 + x) / dx = 1 / (1 + x) = e^-w
                    }
                    gs_wave_sync();
                    if (rank == all - 1) count[wave][t] = had + all;
                }
                gs_wave_sync();
            }
        };
        walk(false);
        __syncthreads();
        // each token's total, its start, and where each wave's part of it begins
        int c = 0;
        if (tid < kTok)
            for (int wv = 0; wv < kSortWaves; wv++) {
                const int x = count[wv][tid];
                count[wv][tid] = c;
                c += x;
            }
        const int inc = (int)gs_wave_incl_scan((uint32_t)c);
        if (lane == 63) wsum[wave] = inc;
        __syncthreads();
        int before = base;
        for (int i = 0; i < wave; i++) before += wsum[i];
        if (tid < kTok) start[tid] = before + inc - c;
        if (tid < kTok && t0 + tid < length) first[b * (length + 1) + t0 + tid] = before + inc - c;
        int total = 0;
        for (int i = 0; i < 16; i++) total += wsum[i];
        __syncthreads();
        walk(true);
        base += total;
        __syncthreads();
    }
    if (tid == 0) first[b * (length + 1) + length] = base;
}

// out[row] = sum over the row's entries of entry_g * W[entry_v]: one workgroup per token, the waves take entries in
// turn and are added in order.
template <int HT>
__global__ __launch_bounds__(256) void k_entries_hidden(const void *weight, int64_t wr, int64_t wd, int wvec, const float *entry_g,
                                                        const int *entry_v, const int *first, int vocab, int length, int dim,
                                                        typename HVal<HT>::t *out) {
    using T = typename HVal<HT>::t;
    __shared__ f32x4 red[3][64];
    const int lane = gs_lane(), wave = threadIdx.x >> 6;
    const int64_t row = blockIdx.x, b = row / length, t = row % length;
    const int lo = first[b * (length + 1) + t], hi = first[b * (length + 1) + t + 1];
    const float *g = entry_g + b * vocab;
    const int *ev = entry_v + b * vocab;
    const bool vec = (dim & 3) == 0;
    for (int d0 = 0; d0 < dim; d0 += 256) {
        const int d = d0 + lane * 4;
        f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
        if (d < dim) {
#pragma unroll 4
            for (int e = lo + wave; e < hi; e += 4) {
                const float x = g[e];
                s += x * row4((const T *)weight + (int64_t)ev[e] * wr, wd, d, dim, wvec);
            }
        }
        if (wave) red[wave - 1][lane] = s;
        __syncthreads();
        if (wave == 0 && d < dim) {
            for (int w = 0; w < 3; w++) s += red[w][lane];
            T *to = out + row * dim + d;
            if (vec) store4(to, s);
            else
                for (int e = 0; e < 4; e++)
                    if (d + e < dim) to[e] = (T)s[e];
        }
        __syncthreads();
    }
}

// dW[v] = sum over texts of g' H[text, token], db[v] = sum of g': a workgroup per 16 terms, a wave per 4 of them.
template <int HT>
__global__ __launch_bounds__(256) void k_entries_weight(Source h, const float *grad, const float *weights, const int *tokens,
                                                        int texts, int vocab, typename HVal<HT>::t *dw, void *db, int db_type) {
    using T = typename HVal<HT>::t;
    __shared__ float sg[64][17];
    __shared__ int st[64][17];
    const int lane = gs_lane(), wave = threadIdx.x >> 6, tid = threadIdx.x;
    const int v0 = blockIdx.x * 16;
    const int dim = h.dim;
    const bool vec = (dim & 3) == 0;
    for (int d0 = 0; d0 < dim; d0 += 256) {
        const int d = d0 + lane * 4;
        f32x4 s[4];
        float bs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < 4; u++) s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int b0 = 0; b0 < texts; b0 += 64) {
            __syncthreads();
            for (int x = tid; x < 64 * 16; x += 256) {
                const int b = b0 + (x >> 4), v = v0 + (x & 15);
                const bool in = b < texts && v < vocab;
                const int64_t at = (int64_t)b * vocab + v;
                int t = in ? tokens[at] : -1;
                if (t >= h.length) t = -1;
                st[x >> 4][x & 15] = t;
                sg[x >> 4][x & 15] = t >= 0 ? grad[at] * expf(-weights[at]) : 0.f;
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int v = wave * 4 + u;
                const int t = st[lane][v];
                const float g = sg[lane][v];
                uint64_t left = __ballot(t >= 0);
                while (left) {
                    const int l = __ffsll((unsigned long long)left) - 1;
                    left &= left - 1;
                    const int tl = __builtin_amdgcn_readlane(t, l);
                    const float gl = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, g), l));
                    bs[u] += gl;
                    if (d < dim) s[u] += gl * row4((const T *)h.p + (int64_t)(b0 + l) * h.s0 + (int64_t)tl * h.s1, h.sd, d, dim, h.vec);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int v = v0 + wave * 4 + u;
            if (v >= vocab) continue;
            if (dw && d < dim) {
                T *to = dw + (int64_t)v * dim + d;
                if (vec) store4(to, s[u]);
                else
                    for (int e = 0; e < 4; e++)
                        if (d + e < dim) to[e] = (T)s[u][e];
            }
            if (db && d0 == 0 && lane == 0) {
                if (db_type == GS_H_F32) ((float *)db)[v] = bs[u];
                else if (db_type == GS_H_F16) ((_Float16 *)db)[v] = (_Float16)bs[u];
                else ((__bf16 *)db)[v] = (__bf16)bs[u];
            }
        }
    }
}

// ---------------------------------------------------------------- host

// Tiles: `Large` for whole batches (two workgroups of 4 waves per CU, three stages of 24 KiB, 128 x 64 per wave);
// `Small` where the kept side is at most one tile of 64, and reading the vocabulary is what takes the time.
template <class T, int NP, bool RK, bool CK>
using Large = Tile<T, NP, 256, 128, 2, 2, 3, RK, CK>;
template <class T, int NP, bool RK, bool CK>
using Small = Tile<T, NP, 64, 64, 2, 2, 6, RK, CK>;

int cu_count(int *cus) {
    int dev = 0;
    GS_CHECK_HIP(hipGetDevice(&dev));
    GS_CHECK_HIP(hipDeviceGetAttribute(cus, hipDeviceAttributeMultiprocessorCount, dev));
    return GS_OK;
}

int es_of(int type) { return type == GS_H_F32 ? 4 : 2; }

bool vec_ok(const void *p, int type, int64_t s0, int64_t s1, int64_t sd) {
    return sd == 1 && s0 % 4 == 0 && s1 % 4 == 0 && (uintptr_t)p % (4 * es_of(type)) == 0;
}

int check_head(const gs_vocab_head *h) {
    GS_REQUIRE(h, "head is NULL");
    GS_REQUIRE(h->type == GS_H_F32 || h->type == GS_H_F16 || h->type == GS_H_BF16, "unknown hidden type %d", h->type);
    GS_REQUIRE(h->bias_type == GS_H_F32 || h->bias_type == GS_H_F16 || h->bias_type == GS_H_BF16, "unknown bias type %d",
               h->bias_type);
    GS_REQUIRE(h->texts >= 0 && h->length >= 0, "negative texts or length");
    GS_REQUIRE((int64_t)h->texts * h->length <= (1 << 28), "%lld rows exceed 2^28", (long long)h->texts * h->length);
    GS_REQUIRE(h->dim >= 1 && h->dim <= 32768, "dim=%d outside [1, 32768]", h->dim);
    GS_REQUIRE(h->vocab >= 1 && h->vocab <= (1 << 20), "vocab=%d outside [1, 2^20]", h->vocab);
    return GS_OK;
}

struct Layout {  // of what both losses and term weights keep in memory
    int rows, dimp, planes, vocabp;
    bool w_direct;
};

Layout layout_of(const gs_vocab_head *h) {
    Layout l;
    l.rows = h->texts * h->length;
    l.planes = h->type == GS_H_F32 ? 3 : 1;
    l.dimp = (int)round_up(h->dim, kStep);
    l.vocabp = (int)round_up(h->vocab, kRowPad);
    // the product reads the vocabulary's rows where they are if each is whole 16-byte pieces
    l.w_direct = l.planes == 1 && h->dim % kStep == 0 && h->weight_dim_stride == 1 && h->weight_row_stride % 8 == 0 &&
                 h->weight_row_stride >= h->dim && h->weight_row_stride < (1 << 20) && (uintptr_t)h->weight_d % 16 == 0;
    return l;
}

struct Saved {
    int *n, *rows, *inv, *seg;
    float *bias;
    uint16_t *hidden, *weight;
};

void take_saved(gs_arena &a, const Layout &l, const gs_vocab_head *h, bool seg, Saved *s) {
    s->n = a.take<int>(64);
    s->rows = a.take<int>(l.rows);
    s->inv = seg ? nullptr : a.take<int>(l.rows);
    s->seg = seg ? a.take<int>(l.rows + kRowPad) : nullptr;
    s->bias = a.take<float>(l.vocabp);
    s->hidden = a.take<uint16_t>((size_t)l.rows * l.planes * l.dimp);
    s->weight = l.w_direct ? nullptr : a.take<uint16_t>((size_t)h->vocab * l.planes * l.dimp);
}

Source hidden_source(const gs_vocab_head *h) {
    return Source{h->hidden_d, h->hidden_text_stride, h->hidden_row_stride, h->hidden_dim_stride, h->length > 0 ? h->length : 1,
                  h->dim, vec_ok(h->hidden_d, h->type, h->hidden_text_stride, h->hidden_row_stride, h->hidden_dim_stride)};
}
Source weight_source(const gs_vocab_head *h) {
    return Source{h->weight_d, 0, h->weight_row_stride, h->weight_dim_stride, 0x7FFFFFFF, h->dim,
                  vec_ok(h->weight_d, h->type, 0, h->weight_row_stride, h->weight_dim_stride)};
}

Operand hidden_operand(const Layout &l, const Saved &s) {
    return Operand{s.hidden, (int64_t)l.planes * l.dimp, l.dimp, (int64_t)l.planes * l.dimp};
}
Operand weight_operand(const Layout &l, const Saved &s, const gs_vocab_head *h) {
    if (l.w_direct) return Operand{(const uint16_t *)h->weight_d, h->weight_row_stride, 0, l.dimp};
    return Operand{s.weight, (int64_t)l.planes * l.dimp, l.dimp, (int64_t)l.planes * l.dimp};
}

int pack_rows(const gs_vocab_head *h, const Source &src, const int *rows, const int *n_d, int n, int dimp, uint16_t *out,
              hipStream_t s) {
    if (n <= 0) return GS_OK;
    const unsigned g = gs_blocks(n, 4, 8192);
    switch (h->type) {
        case GS_H_F32: hipLaunchKernelGGL((k_pack<GS_H_F32, 3>), dim3(g), dim3(256), 0, s, src, rows, n_d, n, dimp, out); break;
        case GS_H_F16: hipLaunchKernelGGL((k_pack<GS_H_F16, 1>), dim3(g), dim3(256), 0, s, src, rows, n_d, n, dimp, out); break;
        default: hipLaunchKernelGGL((k_pack<GS_H_BF16, 1>), dim3(g), dim3(256), 0, s, src, rows, n_d, n, dimp, out); break;
    }
    GS_CHECK_LAUNCH();
    return GS_OK;
}

// Kept rows, bias, hidden states and (where needed) vocabulary rows in the product's form.
int prepare(const gs_vocab_head *h, const Layout &l, const uint8_t *keep, const Saved &sv, hipStream_t s) {
    hipLaunchKernelGGL(k_kept_rows, dim3(1), dim3(1024), 0, s, keep, l.rows, h->length > 0 ? h->length : 1, sv.rows, sv.inv,
                       sv.seg, sv.n);
    GS_CHECK_LAUNCH();
    hipLaunchKernelGGL(k_bias, dim3(gs_blocks(l.vocabp, 256)), dim3(256), 0, s, h->bias_d, h->bias_type, h->vocab, l.vocabp,
                       sv.bias);
    GS_CHECK_LAUNCH();
    if (int rc = pack_rows(h, hidden_source(h), sv.rows, sv.n, l.rows, l.dimp, sv.hidden, s)) return rc;
    if (!l.w_direct)
        if (int rc = pack_rows(h, weight_source(h), nullptr, nullptr, h->vocab, l.dimp, sv.weight, s)) return rc;
    return GS_OK;
}

// f.template operator()<T, NP>() for the head's type
#define GSV_BY_TYPE(type, CALL)                  \
    switch (type) {                              \
        case GS_H_F32: CALL(Bf16, 3); break;     \
        case GS_H_F16: CALL(F16, 1); break;      \
        default: CALL(Bf16, 1); break;           \
    }

constexpr int kSmallRows = 64;

// ---------------------------------------------------------------- losses

struct LossPlan {
    Layout l;
    int top, small;
    int piece, pieces;     // terms per piece (a multiple of kRowPad)
    int row_block;         // terms per softmax-sum block
    int h_tr, h_bc, h_most, slots;
    int64_t part_rows;     // rows of dH parts
};

LossPlan loss_plan(const gs_vocab_head *h, const gs_vocab_targets *t, int cus) {
    LossPlan p;
    p.l = layout_of(h);
    p.top = t->teacher_ids_d ? t->top : 1;
    p.small = p.l.rows <= kSmallRows;
    const int64_t per = (int64_t)(p.l.rows > 0 ? p.l.rows : 1) * p.l.planes * 2;
    int64_t most = (int64_t)kPieceBytes / per / kRowPad * kRowPad;
    if (most < kRowPad) most = kRowPad;
    p.pieces = (int)((p.l.vocabp + most - 1) / most);
    p.piece = (int)round_up((p.l.vocabp + p.pieces - 1) / p.pieces, kRowPad);
    p.pieces = (p.l.vocabp + p.piece - 1) / p.piece;
    p.row_block = p.small ? 32 : 128;
    p.h_tr = (h->dim + (p.small ? 63 : 255)) / (p.small ? 64 : 256);
    p.h_bc = p.small ? 64 : 128;
    p.slots = 2 * cus;
    p.h_most = p.piece / kStep / 8;
    if (p.h_most < 1) p.h_most = 1;
    // split(n) * n, split = slots / (h_tr * ceil(n / bc)): at most slots * bc / h_tr rows, or n
    const int64_t wide = (int64_t)p.slots * p.h_bc / p.h_tr;
    p.part_rows = p.l.rows > wide ? p.l.rows : wide;
    return p;
}

struct LossSaved {
    Saved s;
    float *lse2, *loss;
    int *ids;
    float *share, *ent;
};

void take_loss_saved(gs_arena &a, const LossPlan &p, const gs_vocab_head *h, const gs_vocab_targets *t, LossSaved *s) {
    take_saved(a, p.l, h, false, &s->s);
    s->lse2 = a.take<float>(p.l.rows);
    s->loss = a.take<float>(p.l.rows);
    s->ids = a.take<int>((size_t)p.l.rows * p.top);
    s->share = t->teacher_ids_d ? a.take<float>((size_t)p.l.rows * p.top) : nullptr;
    s->ent = t->teacher_ids_d ? a.take<float>(p.l.rows) : nullptr;
}

struct LossScratch {
    uint8_t *keep;
    float *target;
    float2 *part;
};
void take_loss_scratch(gs_arena &a, const LossPlan &p, LossScratch *s) {
    s->keep = a.take<uint8_t>(p.l.rows);
    s->target = a.take<float>(p.l.rows);
    s->part = a.take<float2>((size_t)(p.l.vocabp / p.row_block) * p.l.rows);
}

struct GradScratch {
    float *factor, *scale, *sums, *part;
    uint16_t *first, *dl;
    int64_t sum_rows;
};
void take_grad_scratch(gs_arena &a, const LossPlan &p, GradScratch *s) {
    const int bc = p.small ? 64 : 128;
    s->factor = a.take<float>(p.l.rows);
    s->scale = a.take<float>(64);
    s->sum_rows = (p.l.rows + bc - 1) / bc * 2;
    s->sums = a.take<float>((size_t)s->sum_rows * p.l.vocabp);
    s->part = a.take<float>((size_t)p.part_rows * p.l.dimp);
    s->first = p.top > 1 ? a.take<uint16_t>((size_t)(p.l.vocabp / kRowPad + 1) * p.l.rows) : nullptr;
    s->dl = a.take<uint16_t>((size_t)p.l.rows * p.l.planes * p.piece);
}

int check_targets(const gs_vocab_head *h, const gs_vocab_targets *t) {
    GS_REQUIRE(t, "targets are NULL");
    GS_REQUIRE((t->targets_d != nullptr) != (t->teacher_ids_d != nullptr), "targets or a teacher's ids, not both or neither");
    if (t->teacher_ids_d) {
        GS_REQUIRE(t->teacher_logits_d, "teacher ids without logits");
        GS_REQUIRE(t->top >= 1 && t->top <= kMaxTop, "top=%d outside [1, %d]", t->top, kMaxTop);
        GS_REQUIRE(t->teacher_type == GS_H_F32 || t->teacher_type == GS_H_F16 || t->teacher_type == GS_H_BF16,
                   "unknown teacher type %d", t->teacher_type);
        GS_REQUIRE(t->temperature > 0.f && t->temperature < INFINITY, "temperature=%g must be positive and finite",
                   (double)t->temperature);
    }
    return GS_OK;
}

float tau_of(const gs_vocab_targets *t) { return t->teacher_ids_d ? t->temperature : 1.f; }

// The tiles' k loop over a [k][x] operand moves its buffer by whole rows, so one row of logit gradients must stay
// within a buffer's 2 GiB with its 32 rows: 32 rows * planes * piece * 2 bytes <= 2^31 holds for every piece here.

template <class T, int NP>
int run_sums(const gs_vocab_head *h, const LossPlan &p, const LossSaved &s, float2 *part, float scale, int cus, hipStream_t st) {
    const Dims d{h->vocab, p.l.rows, p.l.dimp, s.s.n, 0, 1, 0, 1, 0, 0};
    const Operand w = weight_operand(p.l, s.s, h), hid = hidden_operand(p.l, s.s);
    const EpiSums e{s.s.bias, scale, part, p.l.rows};
    if (p.small) return launch_product<Small<T, NP, false, false>>(w, hid, d, e, cus, st);
    return launch_product<Large<T, NP, false, false>>(w, hid, d, e, cus, st);
}

template <class T, int NP, class O>
int run_grad(const gs_vocab_head *h, const LossPlan &p, const LossSaved &s, const GradScratch &g, float scale, bool dh, bool dw,
             bool db, void *dw_d, int cus, hipStream_t st) {
    using S = typename T::store_t;
    const Operand w = weight_operand(p.l, s.s, h), hid = hidden_operand(p.l, s.s);
    const Operand dl{g.dl, (int64_t)NP * p.piece, p.piece, (int64_t)NP * p.piece};
    for (int c = 0; c < p.pieces; c++) {
        const int v0 = c * p.piece, nv = min(p.piece, h->vocab - v0);
        if (nv <= 0) break;
        Operand wp = w;
        wp.p += (int64_t)v0 * w.stride;
        const EpiLogitGrad<S> e{s.s.bias, scale, s.lse2, g.factor, s.s.rows, s.ids, s.share, g.first, p.l.rows, p.top, v0,
                                g.dl, dl.stride, p.piece, db ? g.sums : nullptr, p.l.vocabp};
        const Dims de{nv, p.l.rows, p.l.dimp, s.s.n, 0, 1, 0, 1, 0, 0};
        int rc = p.small ? launch_product<Small<T, NP, false, false>>(wp, hid, de, e, cus, st)
                         : launch_product<Large<T, NP, false, false>>(wp, hid, de, e, cus, st);
        if (rc) return rc;
        if (dh) {
            const EpiHiddenPart eh{g.part, p.l.dimp, c > 0};
            const Dims dd{h->dim, p.l.rows, nv, s.s.n, 0, 1, 0, 0, p.slots, p.h_most};
            rc = p.small ? launch_product<Small<T, NP, true, false>>(wp, dl, dd, eh, cus, st)
                         : launch_product<Large<T, NP, true, false>>(wp, dl, dd, eh, cus, st);
            if (rc) return rc;
        }
        if (dw) {
            const EpiWeightGrad<O> ew{(O *)dw_d + (int64_t)v0 * h->dim, g.scale, h->dim, h->dim % 4 == 0};
            const Dims dd{h->dim, nv, p.l.rows, s.s.n, 0, 0, 1, 1, 0, 0};
            rc = p.small ? launch_product<Small<T, NP, true, true>>(hid, dl, dd, ew, cus, st)
                         : launch_product<Large<T, NP, true, true>>(hid, dl, dd, ew, cus, st);
            if (rc) return rc;
        }
    }
    return GS_OK;
}

}  // namespace gsv

using namespace gsv;

extern "C" int gs_vocab_loss_workspace(const gs_vocab_head *h, const gs_vocab_targets *t, size_t *saved_bytes,
                                       size_t *scratch_bytes, size_t *grad_bytes) {
    if (int rc = check_head(h)) return rc;
    if (int rc = check_targets(h, t)) return rc;
    GS_REQUIRE(saved_bytes && scratch_bytes && grad_bytes, "NULL size pointer");
    int cus = 256;
    if (int rc = cu_count(&cus)) return rc;
    const LossPlan p = loss_plan(h, t, cus);
    LossSaved s;
    LossScratch x;
    GradScratch g;
    gs_arena a{nullptr, 0, 0}, b{nullptr, 0, 0}, c{nullptr, 0, 0};
    take_loss_saved(a, p, h, t, &s);
    take_loss_scratch(b, p, &x);
    take_grad_scratch(c, p, &g);
    *saved_bytes = a.used + 256, *scratch_bytes = b.used + 256, *grad_bytes = c.used + 256;
    return GS_OK;
}

extern "C" int gs_vocab_loss(const gs_vocab_head *h, const gs_vocab_targets *t, int32_t reduction, float *loss_d, void *saved_d,
                             size_t saved_bytes, void *scratch_d, size_t scratch_bytes, void *stream) {
    if (int rc = check_head(h)) return rc;
    if (int rc = check_targets(h, t)) return rc;
    GS_REQUIRE(reduction >= GS_REDUCE_NONE && reduction <= GS_REDUCE_SUM, "unknown reduction %d", reduction);
    int cus = 256;
    if (int rc = cu_count(&cus)) return rc;
    const LossPlan p = loss_plan(h, t, cus);
    LossSaved sv;
    LossScratch x;
    gs_arena a{(char *)saved_d, 0, saved_bytes}, b{(char *)scratch_d, 0, scratch_bytes};
    take_loss_saved(a, p, h, t, &sv);
    take_loss_scratch(b, p, &x);
    if (!a.ok() || !b.ok()) {
        gs_set_error("vocab_loss workspace too small: need %zu + %zu bytes, got %zu + %zu", a.used, b.used, saved_bytes,
                     scratch_bytes);
        return GS_ENOSPC;
    }
    const hipStream_t s = gs_stream(stream);
    const int rows = p.l.rows;
    const float tau = tau_of(t);
    if (reduction == GS_REDUCE_NONE && rows > 0) {
        hipLaunchKernelGGL(k_fill, dim3(gs_blocks(rows, 256, 1024)), dim3(256), 0, s, loss_d, (int64_t)rows, 0.f);
        GS_CHECK_LAUNCH();
    }
    if (rows > 0) {
        if (t->teacher_ids_d) {
            const int th = t->top <= 64 ? 64 : t->top <= 128 ? 128 : 256;
            hipLaunchKernelGGL(k_teacher, dim3(rows), dim3(th), 0, s, t->teacher_ids_d, t->teacher_logits_d, t->teacher_type,
                               t->top, h->vocab, 1.f / tau, sv.ids, sv.share, sv.ent, x.keep);
        } else {
            hipLaunchKernelGGL(k_targets, dim3(gs_blocks(rows, 256)), dim3(256), 0, s, t->targets_d, t->ignore_index, rows,
                               h->vocab, sv.ids, x.keep);
        }
        GS_CHECK_LAUNCH();
    }
    if (int rc = prepare(h, p.l, x.keep, sv.s, s)) return rc;
    if (rows > 0) {
        const Source hs = hidden_source(h), ws = weight_source(h);
        const unsigned g = gs_blocks(rows, 4, 4096);
#define GSV_TL(HT)                                                                                                        \
    hipLaunchKernelGGL((k_target_logits<HT>), dim3(g), dim3(256), 0, s, hs, h->weight_d, h->weight_row_stride,             \
                       h->weight_dim_stride, ws.vec, sv.s.bias, sv.ids, sv.share, p.top, sv.s.rows, sv.s.n, x.target)
        if (h->type == GS_H_F32) GSV_TL(GS_H_F32);
        else if (h->type == GS_H_F16) GSV_TL(GS_H_F16);
        else GSV_TL(GS_H_BF16);
#undef GSV_TL
        GS_CHECK_LAUNCH();
        int rc = GS_OK;
#define GSV_SUMS(T, NP) rc = run_sums<T, NP>(h, p, sv, x.part, kLog2e / tau, cus, s)
        GSV_BY_TYPE(h->type, GSV_SUMS)
#undef GSV_SUMS
        if (rc) return rc;
        const int row_tile = p.small ? 64 : 256;
        const int blocks = (h->vocab + row_tile - 1) / row_tile * (row_tile / p.row_block);
        hipLaunchKernelGGL(k_row_loss, dim3(gs_blocks(rows, 16, 4096)), dim3(256), 0, s, x.part, (int64_t)rows, blocks, sv.s.rows,
                           sv.s.n, x.target, sv.ent, tau, sv.lse2, sv.loss, reduction == GS_REDUCE_NONE ? loss_d : nullptr);
        GS_CHECK_LAUNCH();
    }
    if (reduction != GS_REDUCE_NONE) {
        hipLaunchKernelGGL(k_loss_sum, dim3(1), dim3(1024), 0, s, sv.loss, sv.s.n, reduction == GS_REDUCE_MEAN, loss_d);
        GS_CHECK_LAUNCH();
    }
    return GS_OK;
}

extern "C" int gs_vocab_loss_grad(const gs_vocab_head *h, const gs_vocab_targets *t, int32_t reduction, const float *grad_d,
                                  const void *saved_d, size_t saved_bytes, void *dhidden_d, void *dweight_d, void *dbias_d,
                                  void *scratch_d, size_t scratch_bytes, void *stream) {
    if (int rc = check_head(h)) return rc;
    if (int rc = check_targets(h, t)) return rc;
    GS_REQUIRE(reduction >= GS_REDUCE_NONE && reduction <= GS_REDUCE_SUM, "unknown reduction %d", reduction);
    int cus = 256;
    if (int rc = cu_count(&cus)) return rc;
    const LossPlan p = loss_plan(h, t, cus);
    LossSaved sv;
    GradScratch g;
    gs_arena a{(char *)saved_d, 0, saved_bytes}, b{(char *)scratch_d, 0, scratch_bytes};
    take_loss_saved(a, p, h, t, &sv);
    take_grad_scratch(b, p, &g);
    if (!a.ok() || !b.ok()) {
        gs_set_error("vocab_loss_grad workspace too small: need %zu + %zu bytes, got %zu + %zu", a.used, b.used, saved_bytes,
                     scratch_bytes);
        return GS_ENOSPC;
    }
    const hipStream_t s = gs_stream(stream);
    const int rows = p.l.rows;
    const float tau = tau_of(t);
    hipLaunchKernelGGL(k_row_factor, dim3(1), dim3(1024), 0, s, grad_d, reduction == GS_REDUCE_NONE, sv.s.rows, sv.s.n,
                       reduction == GS_REDUCE_MEAN, tau, h->type == GS_H_F16, g.factor, g.scale);
    GS_CHECK_LAUNCH();
    if (p.top > 1 && rows > 0) {
        hipLaunchKernelGGL(k_entry_starts, dim3(gs_blocks(rows, 64)), dim3(64), 0, s, sv.ids, p.top, sv.s.rows, sv.s.n,
                           p.l.vocabp / kRowPad, kRowPad, (int64_t)rows, g.first);
        GS_CHECK_LAUNCH();
    }
    int rc = GS_OK;
    const float scale = kLog2e / tau;
    // with no rows every launch below is empty of tiles but for dW's, which writes its zeros
    if (rows > 0 || dweight_d) {
        if (h->type == GS_H_F32)
            rc = run_grad<Bf16, 3, float>(h, p, sv, g, scale, dhidden_d, dweight_d, dbias_d, dweight_d, cus, s);
        else if (h->type == GS_H_F16)
            rc = run_grad<F16, 1, _Float16>(h, p, sv, g, scale, dhidden_d, dweight_d, dbias_d, dweight_d, cus, s);
        else
            rc = run_grad<Bf16, 1, __bf16>(h, p, sv, g, scale, dhidden_d, dweight_d, dbias_d, dweight_d, cus, s);
        if (rc) return rc;
    }
    if (dhidden_d && rows > 0) {
        const unsigned gr = gs_blocks(rows, 4, 8192);
#define GSV_HG(O)                                                                                                           \
    hipLaunchKernelGGL((k_hidden_grad<O>), dim3(gr), dim3(256), 0, s, g.part, sv.s.inv, sv.s.n, rows, h->dim, p.l.dimp, p.h_tr, \
                       p.h_bc, p.slots, p.h_most, g.scale, (O *)dhidden_d)
        if (h->type == GS_H_F32) GSV_HG(float);
        else if (h->type == GS_H_F16) GSV_HG(_Float16);
        else GSV_HG(__bf16);
#undef GSV_HG
        GS_CHECK_LAUNCH();
    }
    if (dbias_d) {
        const int bc = p.small ? 64 : 128;
#define GSV_BG(O)                                                                                                            \
    hipLaunchKernelGGL((k_bias_grad<O>), dim3(gs_blocks(h->vocab, 256)), dim3(256), 0, s, g.sums, (int64_t)p.l.vocabp, sv.s.n, bc, \
                       2, h->vocab, g.scale, (O *)dbias_d)
        if (h->bias_type == GS_H_F32) GSV_BG(float);
        else if (h->bias_type == GS_H_F16) GSV_BG(_Float16);
        else GSV_BG(__bf16);
#undef GSV_BG
        GS_CHECK_LAUNCH();
    }
    return GS_OK;
}

// ---------------------------------------------------------------- term weights

extern "C" int gs_term_weights_workspace(const gs_vocab_head *h, int32_t tokens, size_t *bytes, size_t *grad_bytes) {
    if (int rc = check_head(h)) return rc;
    GS_REQUIRE(bytes && grad_bytes, "NULL size pointer");
    const Layout l = layout_of(h);
    gs_arena a{nullptr, 0, 0}, b{nullptr, 0, 0};
    Saved s;
    take_saved(a, l, h, true, &s);
    const size_t n = (size_t)h->texts * h->vocab;
    a.take<char>(n * (tokens ? 8 : 4));
    b.take<float>(n);
    b.take<int>(n);
    b.take<int>((size_t)h->texts * (h->length + 1));
    *bytes = a.used + 256, *grad_bytes = b.used + 256;
    return GS_OK;
}

extern "C" int gs_term_weights(const gs_vocab_head *h, const uint8_t *mask_d, float *weights_d, int32_t *tokens_d,
                               void *workspace_d, size_t workspace_bytes, void *stream) {
    if (int rc = check_head(h)) return rc;
    int cus = 256;
    if (int rc = cu_count(&cus)) return rc;
    const Layout l = layout_of(h);
    gs_arena a{(char *)workspace_d, 0, workspace_bytes};
    Saved sv;
    take_saved(a, l, h, true, &sv);
    const int64_t n = (int64_t)h->texts * h->vocab;
    const int64_t words = tokens_d ? 2 * n : n;
    float *best = a.take<float>(words);
    if (!a.ok()) {
        gs_set_error("term_weights workspace too small: need %zu bytes, got %zu", a.used, workspace_bytes);
        return GS_ENOSPC;
    }
    if (n == 0) return GS_OK;
    const hipStream_t s = gs_stream(stream);
    hipLaunchKernelGGL(k_fill, dim3(gs_blocks(words, 256, 4096)), dim3(256), 0, s, best, words, 0.f);
    GS_CHECK_LAUNCH();
    if (l.rows > 0) {
        // seg is read a whole tile at a time: -1 past the kept rows
        hipLaunchKernelGGL(k_fill, dim3(gs_blocks(l.rows + kRowPad, 256, 1024)), dim3(256), 0, s, (float *)sv.seg,
                           (int64_t)l.rows + kRowPad, __builtin_bit_cast(float, 0xFFFFFFFFu));
        GS_CHECK_LAUNCH();
        if (int rc = prepare(h, l, mask_d, sv, s)) return rc;
        const Dims d{l.rows, h->vocab, l.dimp, sv.n, 1, 0, 0, 1, 0, 0};
        const Operand hid = hidden_operand(l, sv), w = weight_operand(l, sv, h);
        int rc = GS_OK;
#define GSV_MAX(T, NP)                                                                                                    \
    if (tokens_d) {                                                                                                       \
        const EpiTextMax<true> e{sv.bias, sv.seg, best, h->vocab};                                                        \
        rc = l.rows <= kSmallRows ? launch_product<Small<T, NP, false, false>>(hid, w, d, e, cus, s)                      \
                                  : launch_product<Large<T, NP, false, false>>(hid, w, d, e, cus, s);                     \
    } else {                                                                                                              \
        const EpiTextMax<false> e{sv.bias, sv.seg, best, h->vocab};                                                       \
        rc = l.rows <= kSmallRows ? launch_product<Small<T, NP, false, false>>(hid, w, d, e, cus, s)                      \
                                  : launch_product<Large<T, NP, false, false>>(hid, w, d, e, cus, s);                     \
    }
        GSV_BY_TYPE(h->type, GSV_MAX)
#undef GSV_MAX
        if (rc) return rc;
    }
    const unsigned g = gs_blocks(n, 256, 8192);
    const int length = h->length > 0 ? h->length : 1;
    if (tokens_d)
        hipLaunchKernelGGL(k_term_weights<true>, dim3(g), dim3(256), 0, s, best, n, h->vocab, sv.rows, length, weights_d, tokens_d);
    else
        hipLaunchKernelGGL(k_term_weights<false>, dim3(g), dim3(256), 0, s, best, n, h->vocab, sv.rows, length, weights_d, tokens_d);
    GS_CHECK_LAUNCH();
    return GS_OK;
}

extern "C" int gs_term_weights_grad(const gs_vocab_head *h, const float *grad_d, const float *weights_d, const int32_t *tokens_d,
                                    void *dhidden_d, void *dweight_d, void *dbias_d, void *workspace_d, size_t workspace_bytes,
                                    void *stream) {
    if (int rc = check_head(h)) return rc;
    gs_arena a{(char *)workspace_d, 0, workspace_bytes};
    const size_t n = (size_t)h->texts * h->vocab;
    float *entry_g = a.take<float>(n);
    int *entry_v = a.take<int>(n);
    int *first = a.take<int>((size_t)h->texts * (h->length + 1));
    if (!a.ok()) {
        gs_set_error("term_weights_grad workspace too small: need %zu bytes, got %zu", a.used, workspace_bytes);
        return GS_ENOSPC;
    }
    const hipStream_t s = gs_stream(stream);
    const int rows = h->texts * h->length;
    const Source ws = weight_source(h), hs = hidden_source(h);
    if (dhidden_d && rows > 0) {
        hipLaunchKernelGGL(k_sort_entries, dim3(h->texts), dim3(1024), 0, s, grad_d, weights_d, tokens_d, h->vocab, h->length,
                           entry_g, entry_v, first);
        GS_CHECK_LAUNCH();
#define GSV_EH(HT)                                                                                                         \
    hipLaunchKernelGGL((k_entries_hidden<HT>), dim3(rows), dim3(256), 0, s, h->weight_d, h->weight_row_stride,              \
                       h->weight_dim_stride, ws.vec, entry_g, entry_v, first, h->vocab, h->length, h->dim,                  \
                       (typename HVal<HT>::t *)dhidden_d)
        if (h->type == GS_H_F32) GSV_EH(GS_H_F32);
        else if (h->type == GS_H_F16) GSV_EH(GS_H_F16);
        else GSV_EH(GS_H_BF16);
#undef GSV_EH
        GS_CHECK_LAUNCH();
    }
    if (dweight_d || dbias_d) {
#define GSV_EW(HT)                                                                                                         \
    hipLaunchKernelGGL((k_entries_weight<HT>), dim3((h->vocab + 15) / 16), dim3(256), 0, s, hs, grad_d, weights_d, tokens_d, \
                       h->texts, h->vocab, (typename HVal<HT>::t *)dweight_d, dbias_d, h->bias_type)
        if (h->type == GS_H_F32) GSV_EW(GS_H_F32);
        else if (h->type == GS_H_F16) GSV_EW(GS_H_F16);
        else GSV_EW(GS_H_BF16);
#undef GSV_EW
        GS_CHECK_LAUNCH();
    }
    return GS_OK;
}
