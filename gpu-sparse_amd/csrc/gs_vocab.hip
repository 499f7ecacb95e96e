// The vocabulary head of a learned sparse encoder: l = h W^T + b over the vocabulary, with
//   gs_term_weights   w[b][v] = log(1 + relu(max over a text's kept tokens of l)), and its gradient
//   gs_term_weights8  the same of a vocabulary in 8 bits (gs_int8.h)
//   gs_vocab_loss     softmax cross entropy, or distillation from a teacher's top logits, and their gradients
// The logits are made tile by tile (gs_vocab_gemm.h) and consumed in registers.  The losses' gradients make them
// again, a piece of the vocabulary at a time, as gradients in 16 bits that two more products read.
#include <math.h>

#include "gs_int8.h"

namespace gsv {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr int kRowPad = 256;           // rows of the vocabulary are padded to this (bias -inf beyond the last)
constexpr int kMaxTop = 1024;          // teacher logits per row
constexpr size_t kPieceBytes = 1u << 30;  // logit gradients held at a time

// ---------------------------------------------------------------- values

template <class T>
__device__ __forceinline__ uint16_t bits16(float x) {
    return __builtin_bit_cast(uint16_t, (T)x);
}

// Values as bf16 planes, each the nearest to what is left.  One beyond the largest bf16 value takes that for its first, not the
// infinity that is nearer.  An infinity is (+-1, 0, +-inf): a third plane meets first planes alone, which are 0 where their
// value is and else have its sign, so that the pair makes the infinity (or NaN) of an fp32 product, and the other pairs
// finite values that it swallows; as a first plane it would meet 0 and either sign in the other planes.  (Such values are
// looked for together: one by one they cost a loss of 77 rows 7 us of 202.)
template <int N>
__device__ __forceinline__ void split3(const float (&x)[N], uint16_t (&p)[3][N]) {
    constexpr float most = 0x1.fep127f;  // 0x7F7F
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < N; e++) {
        const __bf16 a = (__bf16)x[e];
        const float r = x[e] - (float)a;
        const __bf16 b = (__bf16)r;
        p[0][e] = __builtin_bit_cast(uint16_t, a);
        p[1][e] = __builtin_bit_cast(uint16_t, b);
        p[2][e] = __builtin_bit_cast(uint16_t, (__bf16)(r - (float)b));
        top = fmaxf(top, fabsf(x[e]));
    }
    if (__builtin_expect(top > most, 0)) {
#pragma unroll
        for (int e = 0; e < N; e++) {
            if (!(fabsf(x[e]) > most)) continue;
            const uint32_t sign = __float_as_uint(x[e]) >> 16 & 0x8000;
            const bool infinite = fabsf(x[e]) == INFINITY;
            const float r = fabsf(x[e]) - most;  // of at most 16 bits
            const __bf16 b = (__bf16)r;
            p[0][e] = sign | (infinite ? 0x3F80 : 0x7F7F);
            p[1][e] = sign | (infinite ? 0 : __builtin_bit_cast(uint16_t, b));
            p[2][e] = infinite ? sign | 0x7F80 : sign ^ __builtin_bit_cast(uint16_t, (__bf16)(r - (float)b));
        }
    }
}

template <class T, int NP>
__device__ __forceinline__ void store_planes4(uint16_t *row, int64_t plane, int d, f32x4 x) {
    if constexpr (NP == 1) {
        *reinterpret_cast<Four<uint16_t> *>(row + d) =
            Four<uint16_t>{{bits16<T>(x[0]), bits16<T>(x[1]), bits16<T>(x[2]), bits16<T>(x[3])}};
    } else {
        const float v[4] = {x[0], x[1], x[2], x[3]};
        uint16_t p[3][4];
        split3(v, p);
#pragma unroll
        for (int i = 0; i < 3; i++)
            *reinterpret_cast<Four<uint16_t> *>(row + i * plane + d) = Four<uint16_t>{{p[i][0], p[i][1], p[i][2], p[i][3]}};
    }
}

// 32 columns of 16 rows in blocks: lane l holds those at 4 (l >> 4) of column blocks a and b of row l & 15.  Lanes of two
// rows of lanes swap halves, so that a lane writes eight columns, those of column block (l >> 4) & 1 from 8 (l >> 5) on, and
// the wave whole lines.
template <class T, int NP>
__device__ __forceinline__ void store_blocks(uint16_t *to, int64_t plane, f32x4 a, f32x4 b) {
    uint16_t x[NP][8];
    const float all[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    if constexpr (NP == 1) {
#pragma unroll
        for (int e = 0; e < 8; e++) x[0][e] = bits16<T>(all[e]);
    } else {
        split3(all, x);
    }
#pragma unroll
    for (int i = 0; i < NP; i++) {
        const auto two = [&](int e) { return (uint32_t)x[i][e] | (uint32_t)x[i][e + 1] << 16; };
        const auto u = __builtin_amdgcn_permlane16_swap(two(0), two(4), false, false);
        const auto v = __builtin_amdgcn_permlane16_swap(two(2), two(6), false, false);
        *reinterpret_cast<uint4 *>(to + i * plane) = make_uint4(u[0], v[0], u[1], v[1]);
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
// The values of lanes l and l ^ D (D 16 or 32), the lower lane's first: the same two in both lanes.
template <class T>
struct Two {
    T a, b;
};
template <int D, class T>
__device__ __forceinline__ Two<T> across(T x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    if constexpr (D == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        return {__builtin_bit_cast(T, (uint32_t)r[0]), __builtin_bit_cast(T, (uint32_t)r[1])};
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        return {__builtin_bit_cast(T, (uint32_t)r[0]), __builtin_bit_cast(T, (uint32_t)r[1])};
    }
}
// The same of two values at once: a's in the lanes where bit log2(D) of the lane is 0, b's in the others.
template <int D, class T>
__device__ __forceinline__ Two<T> across(T a, T b) {
    const uint32_t x = __builtin_bit_cast(uint32_t, a), y = __builtin_bit_cast(uint32_t, b);
    if constexpr (D == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(x, y, false, false);
        return {__builtin_bit_cast(T, (uint32_t)r[0]), __builtin_bit_cast(T, (uint32_t)r[1])};
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
        return {__builtin_bit_cast(T, (uint32_t)r[0]), __builtin_bit_cast(T, (uint32_t)r[1])};
    }
}
// the larger one, NaN if either is
__device__ __forceinline__ float maximum(float a, float b, float c) {
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}
// over the 16 lanes of a row of lanes
__device__ __forceinline__ float sum16(float v) { return dpp_add<0x121>(dpp_add<0x122>(dpp_add<0x124>(dpp_add<0x128>(v)))); }

// ---------------------------------------------------------------- setup

// What decides whether a row is kept: a byte per row (NULL: all are), or a target per row.
struct Keep {
    const uint8_t *mask;
    const int64_t *targets;
    int64_t ignore;
    int vocab;
    int total;
    __device__ __forceinline__ bool row(int64_t r) const {
        if (targets) {
            const int64_t t = targets[min(r, (int64_t)total - 1)];
            return r < total && t >= 0 && t < vocab && t != ignore;
        }
        return r < total && (!mask || mask[min(r, (int64_t)total - 1)] != 0);
    }
};

// rows[i]: the i-th kept row, ascending; inv[row]: its place or -1; *n: how many.  For texts of `length` rows, seg[i]
// is the row's text, -1 for the rest of the last tile, and text_first[b] the first place of a text's rows.  One workgroup of
// 1024; a wave takes 1024 rows a turn, 64 at a time.
__device__ __forceinline__ void kept_rows(const Keep &keep, int length, int *rows, int *inv, int *seg, int *text_first, int *n) {
    __shared__ int part[16];
    const int tid = threadIdx.x, lane = gs_lane(), wave = tid >> 6;
    const double by_length = 1.0 / length;
    int base = 0;
    for (int64_t at = 0; at < keep.total; at += 16384) {
        const int64_t r0 = at + wave * 1024;
        uint64_t kept[16];
        int c = 0;
#pragma unroll
        for (int e = 0; e < 16; e++) {
            kept[e] = __ballot(keep.row(r0 + e * 64 + lane));
            c += __popcll(kept[e]);
        }
        if (lane == 0) part[wave] = c;
        __syncthreads();
        int o = base;
        for (int w = 0; w < 16; w++) {
            if (w < wave) o += part[w];
            base += part[w];
        }
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int64_t r = r0 + e * 64 + lane;
            const bool k = (kept[e] >> lane) & 1;
            const int i = o + __popcll(kept[e] & gs_lanemask_lt());
            if (r < keep.total) {
                const int row = (int)r;
                if (inv) inv[row] = k ? i : -1;
                if (seg) {
                    int text = (int)(row * by_length);  // at most one off
                    text += (text + 1) * length <= row ? 1 : 0;
                    text -= text * length > row ? 1 : 0;
                    if (row == text * length) text_first[text] = i;
                    if (k) seg[i] = text;
                }
                if (k) rows[i] = row;
            }
            o += __popcll(kept[e]);
        }
        __syncthreads();
    }
    if (seg && tid == 0) text_first[keep.total / length] = base;
    if (seg)
        for (int i = base + tid; i < round_up(base, kRowPad); i += 1024) seg[i] = -1;
    if (tid == 0) *n = base;
}

// First launch of a call.  Workgroup 0 lists the kept rows; the others write the bias in fp32 (0 without one, -inf for
// the rows that pad the vocabulary: they drop out of every softmax and maximum) and clear what is added to later.  One
// workgroup's walk is what takes the time: 5 us of 45 rows, 14 of 16384.
__global__ __launch_bounds__(1024) void k_setup(Keep keep, int length, int *rows, int *inv, int *seg, int *text_first, int *n, const void *bias,
                                                int bias_type, int vocab, int padded, float *bias_o, float *zero, int64_t zeros) {
    if (blockIdx.x == 0) {
        kept_rows(keep, length, rows, inv, seg, text_first, n);
        return;
    }
    const int64_t by = (int64_t)(gridDim.x - 1) * 1024, at = (int64_t)(blockIdx.x - 1) * 1024 + threadIdx.x;
    for (int64_t v = at; v < padded; v += by) {
        float x = 0.f;
        if (v >= vocab) x = -INFINITY;
        else if (bias)
            x = bias_type == GS_H_F32 ? ((const float *)bias)[v]
                                      : bias_type == GS_H_F16 ? (float)((const _Float16 *)bias)[v] : (float)((const __bf16 *)bias)[v];
        bias_o[v] = x;
    }
    for (int64_t i = at * 4; i < zeros; i += by * 4) {
        if (i + 3 < zeros) *reinterpret_cast<f32x4 *>(zero + i) = f32x4{0.f, 0.f, 0.f, 0.f};
        else
            for (int e = 0; e < 4 && i + e < zeros; e++) zero[i + e] = 0.f;
    }
}

// ---------------------------------------------------------------- packing

template <int HT, int NP>
__device__ __forceinline__ void pack_row(const Source &s, int row, int dimp, uint16_t *dst, int lane) {
    using T = typename HVal<HT>::t;
    using S = std::conditional_t<HT == GS_H_F16, _Float16, __bf16>;
    const T *src = (const T *)s.p + (int64_t)(row / s.length) * s.s0 + (int64_t)(row % s.length) * s.s1;
    for (int d = lane * 4; d < dimp; d += 256) store_planes4<S, NP>(dst, dimp, d, row4(src, s.sd, d, s.dim, s.vec));
}

// ---------------------------------------------------------------- targets

// A teacher's row: q = softmax(logits / tau) over its ids inside the vocabulary, sorted by id (equal ids stay apart,
// in their order), ids beyond them INT_MAX; sum of q log q.  One workgroup per row; LDS holds the row, where each id counts
// those before it: 8192 rows of 64, 13 us.
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

// A teacher's entries of kept row i (source row `row`), and first[t][i]: the first of them with an id of at least
// t * width, t up to tiles.  One wave.
struct TeacherRows {
    const int *ids;  // NULL: no teacher
    const float *share;
    int top, tiles, width;
    int64_t ld;
    int *ids_o;
    float *share_o;
    uint16_t *first;
    __device__ __forceinline__ void take(int64_t i, int row, int lane, int *lds) const {  // lds: room for a row
        const int64_t from = (int64_t)row * top, to = i * top;
        gs_wave_sync();
        for (int k = lane; k < top; k += 64) {
            const int id = ids[from + k];
            lds[k] = id;
            ids_o[to + k] = id;
            share_o[to + k] = share[from + k];
        }
        gs_wave_sync();
        for (int t = lane; t <= tiles; t += 64) {
            const int v = t * width;
            int lo = 0, hi = top;
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (lds[mid] < v) lo = mid + 1;
                else hi = mid;
            }
            first[t * ld + i] = (uint16_t)lo;
        }
    }
};

// Kept row i's target id, and its logit from the unpacked values in fp32.  One wave.
struct TargetRows {
    const int64_t *targets;  // NULL: none
    const float *bias;
    int *ids;
    float *out;
    template <class T>
    __device__ __forceinline__ void take(int64_t i, int row, int lane, const Source &h, const T *src, const Source &w) const {
        const int id = (int)targets[row];
        const T *wrow = (const T *)w.p + id * w.s1;
        float a = 0.f;
        for (int d = lane * 4; d < h.dim; d += 256) {
            const f32x4 x = row4(src, h.sd, d, h.dim, h.vec), y = row4(wrow, w.sd, d, h.dim, w.vec);
            a = fmaf(x[0], y[0], fmaf(x[1], y[1], fmaf(x[2], y[2], fmaf(x[3], y[3], a))));
        }
        a = wave_sum(a);
        if (lane == 0) {
            out[i] = a + bias[id];
            ids[i] = id;
        }
    }
};

// Second launch of a call, a wave per row: the kept hidden states and, where the product cannot read it in place
// (w_rows > 0), the vocabulary as contiguous 16-bit rows (fp32: three planes), zero to a multiple of kStep values; and the
// kept rows' targets.  Bytes: 77 rows and 30522 terms of 384 fp32 values, 117 MB in 22.7 us (5.2 TB/s).
template <int HT, int NP>
__global__ __launch_bounds__(256) void k_pack(Source h, const int *rows, const int *n_d, uint16_t *h_out, Source w, int w_rows,
                                              uint16_t *w_out, int dimp, TargetRows targets, TeacherRows teacher) {
    using T = typename HVal<HT>::t;
    __shared__ int ids_s[4][kMaxTop];
    const int n = *n_d, lane = gs_lane();
    const int64_t items = (int64_t)n + w_rows + (targets.targets || teacher.ids ? n : 0);
    for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < items; i += (int64_t)gridDim.x * 4) {
        if (i < n) {
            pack_row<HT, NP>(h, rows[i], dimp, h_out + i * (int64_t)NP * dimp, lane);
        } else if (i < (int64_t)n + w_rows) {
            pack_row<HT, NP>(w, (int)(i - n), dimp, w_out + (i - n) * (int64_t)NP * dimp, lane);
        } else {
            const int64_t k = i - n - w_rows;
            const int row = rows[k];
            if (teacher.ids) teacher.take(k, row, lane, ids_s[threadIdx.x >> 6]);
            else targets.take(k, row, lane, h, (const T *)h.p + (int64_t)(row / h.length) * h.s0 + (int64_t)(row % h.length) * h.s1, w);
        }
    }
}

// The same for a vocabulary in 8 bits, which is read where it is: the kept hidden states as 8-bit rows of `dimp` values, and
// their scales.  Where k_setup has listed the kept rows:
template <int HT, bool UNIT>
__global__ __launch_bounds__(256) void k_pack8(Source h, const int *rows, const int *n_d, int dimp, int8_t *out, float *scales) {
    using T = typename HVal<HT>::t;
    const int n = *n_d, lane = gs_lane();
    for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < n; i += (int64_t)gridDim.x * 4) {
        const T *row = source_row<T>(h, rows[i]);
        const float scale = quantize_row<UNIT, 2>(row, row_start<UNIT, 2>(row, h, lane), h, dimp, lane,
                                                  [&](int d, uint2 x) { *reinterpret_cast<uint2 *>(out + i * dimp + d) = x; });
        if (lane == 0) scales[i] = scale * kDown;
    }
}
// And where it has not: a workgroup takes kPackRows rows and counts the kept ones before them in the mask itself (a byte per row,
// from the L2), so that there is one launch for both, and no walk by one workgroup: 64 texts of 256 tokens of 768 values 12 us
// against 24 (11 and 13).  Of more than kPackMost rows those counts would cost what they save.  Workgroups after those write the bias.
constexpr int kPackRows = 16, kPackMost = 1 << 16;
template <int HT, bool UNIT>
__global__ __launch_bounds__(256) void k_setup_pack8(Source h, const uint8_t *mask, int total, int texts, int row_blocks, int dimp, int8_t *out,
                                                     float *scales, int *seg, int *text_first, int *n, const void *bias, int bias_type,
                                                     int vocab, int padded, float *bias_o) {
    using T = typename HVal<HT>::t;
    __shared__ int part[4];
    const int tid = threadIdx.x, lane = gs_lane(), wave = tid >> 6;
    if ((int)blockIdx.x >= row_blocks) {
        const int v = ((int)blockIdx.x - row_blocks) * 256 + tid;
        if (v < padded) bias_o[v] = v < vocab ? bias_at(bias, bias_type, v) : -INFINITY;
        return;
    }
    const int r0 = blockIdx.x * kPackRows, length = h.length;
    const auto is_kept = [&](int r) { return r < total && (!mask || mask[r] != 0); };
    int before = 0;
    if (!mask) {
        before = r0;
    } else {
        int c = 0;
#pragma unroll 4
        for (int r = tid * 16; r < r0; r += 4096) {  // whole pieces: r0 is a multiple of 16
            typedef uint32_t words __attribute__((ext_vector_type(4), aligned(1)));
            const words x = *reinterpret_cast<const words *>(mask + r);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t any = ((x[e] & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) | x[e];  // bit 7 of each byte that is not 0
                c += __popc(any & 0x80808080u);
            }
        }
        c = (int)gs_wave_sum((uint32_t)c);
        if (lane == 0) part[wave] = c;
        __syncthreads();
        before = part[0] + part[1] + part[2] + part[3];
    }
    const uint64_t kept = __ballot(lane < kPackRows && is_kept(min(r0 + lane, total)));
    if (wave == 0 && lane < kPackRows) {
        const int r = r0 + lane, at = before + __popcll(kept & gs_lanemask_lt());
        if (r < total) {
            const int text = r / length;
            if (r == text * length) text_first[text] = at;
            if ((kept >> lane) & 1) seg[at] = text;
        }
    }
    if ((int)blockIdx.x == row_blocks - 1) {
        const int all = before + __popcll(kept);
        if (tid == 0) *n = all, text_first[texts] = all;
        for (int i = all + tid; i < (int)round_up(all, kRowPad); i += 256) seg[i] = -1;
    }
    // a wave's kept rows, one asked for before the one before is done
    RowStart<2, T> x;
    const T *row = nullptr;
    int r = -1;
    for (int in = wave; in < kPackRows + 4; in += 4) {
        const bool on = in < kPackRows && ((kept >> in) & 1);
        if (in < kPackRows && !on) continue;
        const T *row1 = row;
        RowStart<2, T> x1;
        if (on) {
            row1 = source_row<T>(h, r0 + in);
            x1 = row_start<UNIT, 2>(row1, h, lane);
        }
        if (r >= 0) {
            const int at = before + __popcll(kept & ((1ull << r) - 1));
            const float scale = quantize_row<UNIT, 2>(row, x, h, dimp, lane,
                                                      [&](int d, uint2 y) { *reinterpret_cast<uint2 *>(out + (int64_t)at * dimp + d) = y; });
            if (lane == 0) scales[at] = scale * kDown;
        }
        r = in, row = row1, x = x1;
    }
}

// One upstream value for all rows is kept out of the rounding of the logit gradients, so that their largest parts, p - 1
// at a target, are rounded next to 1, where they almost lie; what is summed over them is multiplied with value().  Values
// of their own (one per row) go into the gradients.  fp16's range asks for a power of two `up` as well: |p - share| <= 1, so
// the gradients' largest magnitude is put at 2^11 to 2^12.
struct Upstream {
    const float *grad;
    const int *n;
    int mean;
    float by;            // temperature / up
    const float *scale;  // per-row values: 1 / up, made by k_row_factor
    // 0 where no row counts: sums of nothing stay 0 under an infinite value
    __device__ __forceinline__ float value() const {
        const int rows = *n;
        return rows == 0 ? 0.f : scale ? *scale : *grad * (mean ? by / (float)rows : by);
    }
};

// ---------------------------------------------------------------- epilogues

// The target shares of the kept rows, ascending by id within a row.
struct Entries {
    const int *ids;         // [kept row][top]
    const float *share;
    const uint16_t *first;  // [block of terms + 1][kept row]: a block is what a wave of the losses' tiles holds
    int64_t ld;
    int top;
};

// A wave's part of them: lane l holds those of token n0 + l (of the wave's 16 MC) in the wave's block of terms.  The first
// four are asked for before the tile's last stage (one after the other, column block by column block, they took as long as a
// third of the product).
template <int MR, int MC>
struct Held {
    static constexpr int M = 4;
    const int *ids;
    const float *share;
    int wv, count;
    int id[M];
    float part[M];
    __device__ __forceinline__ Held(const Entries &s, int n0, int n_c, int wv_, int lane) : wv(wv_) {
        const int n = n0 + lane;
        const bool on = lane < 16 * MC && n < n_c;
        const int64_t t = (int64_t)(wv / (16 * MR)) * s.ld + n;
        const int k = on ? s.first[t] : 0;
        count = on ? s.first[t + s.ld] - k : 0;
        ids = s.ids + (int64_t)n * s.top + k;
        share = s.share + (int64_t)n * s.top + k;
#pragma unroll
        for (int m = 0; m < M; m++) {
            id[m] = m < count ? ids[m] : 0;
            part[m] = m < count ? share[m] : 0.f;
        }
    }
    // f(mine, share) for each entry of column block j's tokens: in the lane that holds the entry's term in register
    // `mine` = 4 i + e; other lanes get -1.
    template <class F>
    __device__ __forceinline__ void each(int j, int lane, F &&f) const {
        const int from = 16 * j + (lane & 15), q = lane >> 4;
        const uint64_t block = 0xFFFFull << (16 * j);
        const auto one = [&](int m, int x, float s) {
            if (!(__ballot(m < count) & block)) return false;
            const int lv = __shfl(m < count ? x - wv : -1, from, GS_WAVE);
            const float sh = __shfl(s, from, GS_WAVE);
            f(lv >= 0 && ((lv >> 2) & 3) == q ? (lv >> 4) * 4 + (lv & 3) : -1, sh);
            return true;
        };
#pragma unroll
        for (int m = 0; m < M; m++)
            if (!one(m, id[m], part[m])) return;
        for (int m = M; one(m, m < count ? ids[m] : 0, m < count ? share[m] : 0.f); m++) {
        }
    }
};

struct NoneHeld {
    template <class F>
    __device__ __forceinline__ void each(int, int, F &&) const {}
};
template <class TL, bool SHARES>
__device__ __forceinline__ auto held_of(const Entries &s, const Place &at, int wv) {
    if constexpr (SHARES) return Held<TL::MR, TL::MC>(s, at.col0, at.n_c, wv, at.lane);
    else return NoneHeld{};
}

// Adds the bias of a tile's rows (side array 0) where its sums did not start with it.
template <class TL, class Epi>
__device__ __forceinline__ void add_row_bias(f32x4 (&acc)[TL::MR][TL::MC], const Place &at) {
    if constexpr (!starts_with_rows<TL, Epi>) {
#pragma unroll
        for (int i = 0; i < TL::MR; i++) {
            const f32x4 b = at.side4(0, at.r_in + 16 * i + 4 * (at.lane >> 4));
#pragma unroll
            for (int j = 0; j < TL::MC; j++) acc[i][j] += b;
        }
    }
}

// Softmax sums of a tile: per token the largest scaled logit and the sum of 2^(scaled logit - it), over each wave's
// terms: part[block of terms][token]; with SHARES also the sum of share * logit: dots[block of terms][token].  An exponent
// takes four times an addition's cycles, and two waves' epilogues share a SIMD: a fifth of a tile's time at 768 values.
// 8192 rows, 128003 terms, 1024 values: 1.65 ms (1300 TFLOP/s); 5734 rows, 30522, 768, with entries: 287 us (940).
template <bool SHARES>
struct EpiSums {
    const float *bias;
    float scale;  // log2(e) / temperature
    float2 *part;
    float *dots;
    int64_t ld;
    Entries entries;
    static constexpr int sides = 1;
    static constexpr bool row_bias = true;
    __device__ __forceinline__ SideArray side(int, int r0, int, const Shape &) const { return {bias + r0, 256}; }
    template <class TL>
    __device__ __forceinline__ auto before(const Place &at) const {
        return held_of<TL, SHARES>(entries, at, at.row0);
    }
    template <class TL, class H>
    __device__ __forceinline__ void run(f32x4 (&acc)[TL::MR][TL::MC], const Place &at, const H &held) const {
        const int q = at.lane >> 4;
        add_row_bias<TL, EpiSums>(acc, at);
        const int64_t block = at.row0 / (TL::MR * 16);
#pragma unroll
        for (int j = 0; j < TL::MC; j++) {
            const int n = at.col0 + 16 * j + (at.lane & 15);
            float m = -INFINITY;
#pragma unroll
            for (int i = 0; i < TL::MR; i++) m = maximum(maximum(m, acc[i][j][0], acc[i][j][1]), acc[i][j][2], acc[i][j][3]);
            float mc = m * scale, s = 0.f;
            const float sub = m == -INFINITY ? 0.f : mc;
#pragma unroll
            for (int i = 0; i < TL::MR; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) s += __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], scale, -sub));
            float dot = 0.f;
            if (SHARES)
                held.each(j, at.lane, [&](int mine, float share) {
                    float x = 0.f;
#pragma unroll
                    for (int i = 0; i < TL::MR; i++) {
                        const f32x4 &y = acc[i][j];
                        const float a = mine & 1 ? y[1] : y[0], b = mine & 1 ? y[3] : y[2];
                        x = mine >> 2 == i ? (mine & 2 ? b : a) : x;
                    }
                    if (share != 0.f) dot = fmaf(share, x, dot);  // x is 0 in the lanes without the entry
                });
            const auto join = [&](Two<float> m2, Two<float> s2, Two<float> d2) {
                mc = fmaxf(m2.a, m2.b);
                const float by = mc == -INFINITY ? 0.f : mc;
                s = s2.a * __builtin_amdgcn_exp2f(m2.a - by) + s2.b * __builtin_amdgcn_exp2f(m2.b - by);
                if (SHARES) dot = d2.a + d2.b;
            };
            join(across<16>(mc), across<16>(s), SHARES ? across<16>(dot) : Two<float>{0.f, 0.f});
            join(across<32>(mc), across<32>(s), SHARES ? across<32>(dot) : Two<float>{0.f, 0.f});
            if (q == 0 && n < at.n_c) {
                part[block * ld + n] = make_float2(mc, s);
                if (SHARES) dots[block * ld + n] = dot;
            }
        }
    }
};

// Gradients of a tile's logits: (softmax - target shares) times the row's factor, rounded to 16 bits once (three
// planes for fp32), in blocks, and their sums over each wave's tokens for the bias.  The rounding is what the products that read
// them take; with 32 bits they would be six plane pairs.  It costs, of all gradients against float64: distillation in bf16
// 2.3e-3 where fp32 logit gradients have 1.7e-3, which is the results' own rounding, in fp16 2.9e-4 and 2.1e-4; targets 1.7e-3
// either way.  The rows of a block past the last
// kept row are zeros: dW sums over them.  The products are made a second time rather than kept: 8192 rows of 128003
// logits are 2 GB to write and to read, 0.8 ms, against 1.6 for the product, but in 16 bits they would lose what the losses need.
// 1.79 ms there, in two pieces (1200 TFLOP/s, 2.1 GB written).
template <class S, bool SHARES>
struct EpiLogitGrad {
    const float *bias;
    float scale;
    const float *lse2;     // log2 of the softmax sum, per kept row
    const float *factor;   // per kept row; NULL: `up` for all
    float up, up_log2;     // a power of two
    Entries entries;
    int v0;                // first term of this piece
    uint16_t *out;
    int64_t ld, plane;     // of the blocks, as an Operand's
    float *col_sums;       // NULL: not wanted; [wave's block of tokens][padded vocabulary]
    int64_t sums_ld;
    static constexpr int sides = 4;
    static constexpr bool row_bias = true;
    __device__ __forceinline__ SideArray side(int a, int r0, int c0, const Shape &s) const {
        if (a == 0) return {bias + v0 + r0, 256};
        if (a == 1) return {lse2 + c0, s.nc - c0};
        if (a == 2) return {factor + c0, factor ? s.nc - c0 : 0};
        return {entries.ids + c0, SHARES ? 0 : s.nc - c0};  // one target per row
    }
    template <class TL>
    __device__ __forceinline__ auto before(const Place &at) const {
        return held_of<TL, SHARES>(entries, at, v0 + at.row0);
    }
    template <class TL, class H>
    __device__ __forceinline__ void run(f32x4 (&acc)[TL::MR][TL::MC], const Place &at, const H &held) const {
        const int q = at.lane >> 4;
        f32x4 sums[TL::MR];
#pragma unroll
        for (int i = 0; i < TL::MR; i++) sums[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        add_row_bias<TL, EpiLogitGrad>(acc, at);
        const int wv = v0 + at.row0;  // the wave's first term
        const bool written = at.col0 / kBlock * kBlock < at.n_c;
        uint16_t *to = out + at.col0 / kBlock * ld + (int64_t)(at.row0 / kBlock) * kBlockValues +
                       in_block(at.col0 % kBlock + (at.lane & 15), at.row0 % kBlock + 16 * (q & 1) + 8 * (q >> 1));
#pragma unroll
        for (int j = 0; j < TL::MC; j++) {
            const int n = at.col0 + 16 * j + (at.lane & 15);
            const bool on = n < at.n_c;
            const int in = at.c_in + 16 * j + (at.lane & 15);
            const float l = at.side(1, in) - up_log2;  // 2^(x - l) comes out times up
#pragma unroll
            for (int i = 0; i < TL::MR; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[i][j][e] = __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], scale, -l));
            const auto off = [&](int mine, float share) {
                float by[4];
#pragma unroll
                for (int e = 0; e < 4; e++) by[e] = (mine & 3) == e ? share * up : 0.f;
#pragma unroll
                for (int i = 0; i < TL::MR; i++) {
                    const float here = mine >> 2 == i ? -1.f : 0.f;
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[i][j][e] = fmaf(here, by[e], acc[i][j][e]);
                }
            };
            if constexpr (SHARES) {
                held.each(j, at.lane, off);
            } else {
                const int lv = on ? __float_as_int(at.side(3, in)) - wv : -1;
                const bool here = lv >= 0 && lv < TL::MR * 16;
                if (__any(here)) off(here && ((lv >> 2) & 3) == q ? (lv >> 4) * 4 + (lv & 3) : -1, 1.f);
            }
            if (factor) {
                const float f = at.side(2, in);
#pragma unroll
                for (int i = 0; i < TL::MR; i++) acc[i][j] *= f;
            }
#pragma unroll
            for (int i = 0; i < TL::MR; i++) {
                acc[i][j] = on ? acc[i][j] : f32x4{0.f, 0.f, 0.f, 0.f};
                sums[i] += acc[i][j];
            }
            if (written) {
#pragma unroll
                for (int i = 0; i < TL::MR; i += 2)
                    store_blocks<S, TL::planes>(to + in_block(16 * j, 16 * (i & 3)) + (i >> 2) * kBlockValues, plane, acc[i][j], acc[i + 1][j]);
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

// dW: rows are dim, columns terms; out[term][dim] times *scale.  It and dH, one launch: 8192 rows, 128003 terms, 1024 values
// 4.0 ms (1070 TFLOP/s); 2458 rows, 30522, 768 222 us (1040).  What bounds them: loads that two stages do not hide.
template <class O>
struct EpiWeightGrad {
    O *out;
    Upstream up;
    int dim, vec;
    static constexpr int sides = 0;
    static constexpr bool row_bias = false;
    __device__ __forceinline__ SideArray side(int, int, int, const Shape &) const { return {nullptr, 0}; }
    template <class TL>
    __device__ __forceinline__ NoneHeld before(const Place &) const {
        return {};
    }
    template <class TL>
    __device__ __forceinline__ void run(f32x4 (&acc)[TL::MR][TL::MC], const Place &at, const NoneHeld &) const {
        const float s = up.value();
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
    static constexpr int sides = 0;
    static constexpr bool row_bias = false;
    __device__ __forceinline__ SideArray side(int, int, int, const Shape &) const { return {nullptr, 0}; }
    template <class TL>
    __device__ __forceinline__ NoneHeld before(const Place &) const {
        return {};
    }
    template <class TL>
    __device__ __forceinline__ void run(f32x4 (&acc)[TL::MR][TL::MC], const Place &at, const NoneHeld &) const {
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

// Largest logit of each text and term: rows are kept tokens (ascending by text), columns terms.  A wave's rows are a
// block w of tokens; for each text b in it the largest logits go to slot w + b (along the blocks and texts one of the
// two grows with each pair, so slots are distinct, and those of a text lie one after the other), with TOK also the
// lowest kept row that has it (any number where that is a NaN or -inf).  k_term_weights takes a text's slots together.  The bias is added to the maximum
// (rounding keeps order).  The product bounds it: 10240 rows, 30522 terms, 768 values, 372 us (1290 TFLOP/s); texts of 20 tokens,
// whose maxima are joined across lanes and written seven times a wave: 1280 rows 67 us (890).
//
// Q8: operands in 8 bits.  Sums take their row's scale before they are compared, their column's magnitude after (in_order): 10240 rows, 30522 terms, 768
// values 201 us (2390 TOP/s, what a library product of 16384^3 reaches; the matrix units are busy half of that time).  Tiles are chosen as
// for 16 bits (class_of); us for terms in 30522 columns of 768, by the edge of a tile's rows:
//   rows                   32    64    80   128   160   256   320   512   768
//   texts of 16    64    18.0  18.3  20.2  20.7  24.8  29.0  33.2  42.5  57.9
//                 128    19.1  20.0  20.1  20.9  21.6  22.5  30.4  31.8  40.5
//                 256    22.3  23.1  23.5  24.5  24.7  27.0  27.9  29.8  42.7
//              k_few8    12.8  19.6  25.8
//   texts of 4     64    20.6  21.9  25.4  27.0  32.9  39.9  46.4  60.8  85.2
//                 128    20.9  24.1  24.7  28.2  29.9  32.9  45.0  47.9  63.5
//                 256    23.8  27.0  28.6  33.4  34.4  41.3  42.6  46.2  69.6
//              k_few8    12.3  20.4  25.4
template <bool TOK, bool Q8 = false>
struct EpiTextMax {
    const float *bias;
    const int *seg;   // text of each kept row, -1 for the rest of the last tile
    float *best;      // [slot][vocab]
    int *where;
    int vocab;
    const float *row_scales, *col_scales;  // of Q8; the rows' times kDown
    static constexpr int sides = Q8 ? 4 : 2;
    static constexpr bool row_bias = false;
    __device__ __forceinline__ SideArray side(int a, int r0, int c0, const Shape &s) const {
        if (a == 2) return {row_scales + r0, s.nr - r0};
        if (a == 3) return {col_scales + c0, s.nc - c0};
        return a == 0 ? SideArray{bias + c0, 256} : SideArray{seg + r0, 256};
    }

    // Takes rows row .. row + 3's values into the lane's maximum, and the first row that has it
    __device__ __forceinline__ static void take(f32x4 x, int row, float &top, int &tok) {
        if (TOK) {
            const float m = maximum(maximum(x[0], x[1], x[2]), x[3], x[3]);
            int r = x[2] == m ? row + 2 : row + 3;
            r = x[1] == m ? row + 1 : r;
            r = x[0] == m ? row : r;
            tok = m > top ? r : tok;
            top = maximum(top, m, m);
        } else {
            top = maximum(maximum(top, x[0], x[1]), x[2], x[3]);
        }
    }
    // The column blocks' maxima over the four rows of lanes, each block's in a row of lanes of its own.
    template <int MC>
    __device__ __forceinline__ void flush(int64_t slot, float (&top)[MC], int (&tok)[MC], float b, float by, const Place &at) const {
        static_assert(MC == 2 || MC == 4, "a row of lanes writes one column block");
        const auto join = [&](Two<float> x2, Two<int> r2, float &x, int &r) {
            if (TOK) r = x2.b > x2.a || (x2.b == x2.a && r2.b < r2.a) ? r2.b : r2.a;
            x = maximum(x2.a, x2.b, x2.b);
        };
        float x[MC / 2];
        int r[MC / 2];
#pragma unroll
        for (int j = 0; j < MC; j += 2)
            join(across<16>(top[j], top[j + 1]), TOK ? across<16>(tok[j], tok[j + 1]) : Two<int>{0, 0}, x[j / 2], r[j / 2]);
        float best_x;
        int best_r = 0;
        join(across<32>(x[0], x[MC / 2 - 1]), TOK ? across<32>(r[0], r[MC / 2 - 1]) : Two<int>{0, 0}, best_x, best_r);
        const int v = at.col0 + at.lane;
        if (at.lane < 16 * MC && v < vocab) {
            best[slot * vocab + v] = Q8 ? fmaf(best_x * fabsf(by), kUp, b) : best_x + b;
            if (TOK) where[slot * vocab + v] = best_r;
        }
    }
    template <class TL>
    __device__ __forceinline__ NoneHeld before(const Place &) const {
        return {};
    }
    template <class TL>
    __device__ __forceinline__ void run(f32x4 (&acc)[TL::MR][TL::MC], const Place &at, const NoneHeld &) const {
        const int q = at.lane >> 4;
        if (at.row0 >= at.n_r) return;
        const int64_t block = at.row0 / (TL::MR * 16);
        const float b = at.side(0, at.c_in + (at.lane & (16 * TL::MC - 1)));  // of the column that the lane writes
        const float by = Q8 ? at.side(3, at.c_in + (at.lane & (16 * TL::MC - 1))) : 1.f;
        const bool some = Q8 && __any(reorders(by));
        float top[TL::MC];
        int tok[TL::MC];
#pragma unroll
        for (int j = 0; j < TL::MC; j++) top[j] = -INFINITY, tok[j] = 0x7FFFFFFF;
        int cur = gs_uniform(__float_as_int(at.side(1, at.r_in)));
#pragma unroll
        for (int i = 0; i < TL::MR; i++) {
            const int row = at.row0 + 16 * i + 4 * q;
            const f32x4 sf = at.side4(1, at.r_in + 16 * i + 4 * q);
            const int sv[4] = {__float_as_int(sf[0]), __float_as_int(sf[1]), __float_as_int(sf[2]), __float_as_int(sf[3])};
            const int lo = __builtin_amdgcn_readlane(sv[0], 0), hi = __builtin_amdgcn_readlane(sv[3], 48);
            if (Q8) {
                const f32x4 sc = at.side4(2, at.r_in + 16 * i + 4 * q);
#pragma unroll
                for (int j = 0; j < TL::MC; j++) acc[i][j] = __builtin_convertvector(__builtin_bit_cast(i32x4, acc[i][j]), f32x4) * sc;
                if (__builtin_expect(some, 0)) {
#pragma unroll
                    for (int j = 0; j < TL::MC; j++) {
                        const int c = at.c_in + 16 * j + (at.lane & 15);
                        const ColumnScale col{at.side(3, c), at.side(0, c)};
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[i][j][e] = in_order(acc[i][j][e], col);
                    }
                }
            }
            if (lo == cur && hi == cur) {  // all of one text
#pragma unroll
                for (int j = 0; j < TL::MC; j++) take(acc[i][j], row, top[j], tok[j]);
                continue;
            }
            int now = lo;
            while (now >= 0) {  // rows past the last kept one are -1, and come last
                if (now != cur) {
                    flush<TL::MC>(block + cur, top, tok, b, by, at);
                    cur = now;
#pragma unroll
                    for (int j = 0; j < TL::MC; j++) top[j] = -INFINITY, tok[j] = 0x7FFFFFFF;
                }
                int next = 0x7FFFFFFF;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (sv[e] > now) next = min(next, sv[e]);
#pragma unroll
                for (int j = 0; j < TL::MC; j++) {
                    f32x4 x;
#pragma unroll
                    for (int e = 0; e < 4; e++) x[e] = sv[e] == now ? acc[i][j][e] : -INFINITY;
                    take(x, row, top[j], tok[j]);
                }
                next = min(min(__builtin_amdgcn_readlane(next, 0), __builtin_amdgcn_readlane(next, 16)),
                           min(__builtin_amdgcn_readlane(next, 32), __builtin_amdgcn_readlane(next, 48)));
                now = next == 0x7FFFFFFF ? -1 : next;
            }
        }
        flush<TL::MC>(block + cur, top, tok, b, by, at);
    }
};

// ---------------------------------------------------------------- losses' small kernels

// log2 of each kept row's softmax sum, and its loss.  X rows per 256 threads: 16 read the sums by 128-byte lines, 4 leave
// few rows enough threads (45 rows of 954 sums: 25 -> 8 us).
template <int X>
__global__ __launch_bounds__(256) void k_row_loss(const float2 *part, const float *dots, int64_t ld, int blocks,
                                                  const int *rows, const int *n_d, const float *target, const float *ent, float tau, float *lse2_o,
                                                  float *loss_o, float *loss_rows) {
    constexpr int Y = 256 / X;
    __shared__ float sm[Y][X + 1], ss[Y][X + 1], sd[Y][X + 1];
    const int n = *n_d, x = threadIdx.x % X, y = threadIdx.x / X;
    for (int64_t i0 = (int64_t)blockIdx.x * X; i0 < n; i0 += (int64_t)gridDim.x * X) {
        const int64_t i = i0 + x;
        float m = -INFINITY, s = 0.f, dot = 0.f;
        auto add = [&](float mo, float so) {
            const float mn = fmaxf(m, mo), by = mn == -INFINITY ? 0.f : mn;
            s = s * __builtin_amdgcn_exp2f(m - by) + so * __builtin_amdgcn_exp2f(mo - by);
            m = mn;
        };
        if (i < n) {
#pragma unroll 4
            for (int b = y; b < blocks; b += Y) {
                const float2 p = part[b * ld + i];
                if (dots) dot += dots[b * ld + i];
                add(p.x, p.y);
            }
        }
        sm[y][x] = m, ss[y][x] = s, sd[y][x] = dot;
        __syncthreads();
        for (int by = Y / 2; by > 0; by >>= 1) {  // joined in a tree
            if (y < by) {
                add(sm[y + by][x], ss[y + by][x]);
                dot += sd[y + by][x];
                sm[y][x] = m, ss[y][x] = s, sd[y][x] = dot;
            }
            __syncthreads();
        }
        if (y == 0 && i < n) {
            const float l2 = m + log2f(s);
            const int row = rows[i];
            const float loss = tau * tau * ((ent ? ent[row] : 0.f) + (l2 * kLn2 - (target ? target[i] : dot) / tau));
            lse2_o[i] = l2;
            loss_o[i] = loss;
            if (loss_rows) loss_rows[row] = loss;
        }
        __syncthreads();
    }
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

// Upstream values of their own for the kept rows, times the temperature.  fp16: one power of two for all of them (`scale`
// undoes it), and where they spread by more than 2^4 one for each row's own (`own`), with which the logit gradients are made
// a second time, for dH: of n_own[0] rows, while dH of the first ones is of n_own[1] (4099 rows of 768, 30522 terms: 885 us,
// spread 1090).  Next to 2^11 even the mean probability of 2^20 terms stays among fp16's normal numbers,
// next to 2^-4 of that too, but rows of smaller values would lose theirs (dW and db, sums over rows, lose nothing next to the
// largest's).  undo[i] gives dH's row back.
struct RowFactors {
    float *factor, *scale;
    float *own, *undo;  // fp16 alone
    int *n_own;
};
__global__ __launch_bounds__(1024) void k_row_factor(const float *grad, const int *rows, const int *n_d, float tau, RowFactors o) {
    __shared__ float part[2][16];
    const int n = *n_d;
    float most = 0.f, least = INFINITY;
    for (int i = threadIdx.x; i < n; i += 1024) {
        const float f = grad[rows[i]] * tau, a = fabsf(f);
        o.factor[i] = f;
        most = fmaxf(most, a);
        if (a > 0.f) least = fminf(least, a);
    }
    float up = 1.f;
    if (o.own) {
        most = wave_max(most), least = -wave_max(-least);
        if (gs_lane() == 0) part[0][threadIdx.x >> 6] = most, part[1][threadIdx.x >> 6] = least;
        __syncthreads();
        most = part[0][0], least = part[1][0];
        for (int w = 1; w < 16; w++) most = fmaxf(most, part[0][w]), least = fminf(least, part[1][w]);
        const bool in_range = most > 0.f && most < 3e38f, spread = in_range && least < most * 0.0625f;
        if (in_range) up = ldexpf(1.f, max(-120, min(120, 11 - ilogbf(most))));
        for (int i = threadIdx.x; i < n; i += 1024) {
            const float f = o.factor[i];
            const int e = fabsf(f) > 0.f && fabsf(f) < INFINITY ? ilogbf(f) : 11;  // 0 and NaN as they are
            o.own[i] = ldexpf(f, 11 - e);
            o.undo[i] = spread ? ldexpf(1.f, e - 11) : 1.f / up;
            o.factor[i] = f * up;
        }
        if (threadIdx.x == 0) o.n_own[0] = spread ? n : 0, o.n_own[1] = spread ? 0 : n;
    }
    if (threadIdx.x == 0) *o.scale = 1.f / up;
}

// The bias's gradient: the tiles' column sums added up in order.  `blocks` of them.
struct BiasSums {
    const float *sums;  // NULL: not wanted
    int64_t ld;
    int edge, waves;    // tokens of a tile, sums of one
    int vocab, type;
    void *out;
};

// Last launch of a gradient.  dH of every source row from its parts (0 for rows that are not kept): with few rows, and so
// many parts, a workgroup of W = 16 waves takes 256 values of a row, the waves take parts in turn and are added in order; else
// (W = 4) a wave does.  undo: a row's own scale, NULL: the upstream value's.  Then workgroups of 32 terms of the bias.
// Bytes: 8192 rows of 1024 values, 54 us.
template <class O, int W>
__global__ __launch_bounds__(64 * W) void k_finish_grad(const float *part, const int *inv, const int *n_d, const int *parts_d,
                                                        int total, int dim, int dimp, Upstream up, const float *undo, O *out,
                                                        int hidden_blocks, BiasSums bias) {
    __shared__ f32x4 red[W][64];
    const int n = *n_d, lane = gs_lane(), wave = threadIdx.x >> 6;
    const float s = up.value();
    if ((int)blockIdx.x >= hidden_blocks) {
        constexpr int Y = 2 * W;
        float *const sum = reinterpret_cast<float *>(red);  // [Y][32]
        const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
        const int v = ((int)blockIdx.x - hidden_blocks) * 32 + x;
        const int blocks = (n + bias.edge - 1) / bias.edge * bias.waves;
        float t = 0.f;
        if (v < bias.vocab) {
#pragma unroll 4
            for (int b = y; b < blocks; b += Y) t += bias.sums[b * bias.ld + v];
        }
        sum[y * 32 + x] = t;
        __syncthreads();
        if (y == 0 && v < bias.vocab) {
            for (int i = 1; i < Y; i++) t += sum[i * 32 + x];
            t *= s;
            if (bias.type == GS_H_F32) ((float *)bias.out)[v] = t;
            else if (bias.type == GS_H_F16) ((_Float16 *)bias.out)[v] = (_Float16)t;
            else ((__bf16 *)bias.out)[v] = (__bf16)t;
        }
        return;
    }
    const int parts = *parts_d;
    const bool vec = (dim & 3) == 0;
    const int chunks = (dim + 255) / 256;
    const auto put = [&](int64_t r, int i, int d, f32x4 x) {
        x *= i < 0 ? 0.f : undo ? undo[i] : s;  // an infinite value leaves rows that are not kept 0
        O *to = out + r * dim + d;
        if (vec) store4(to, x);
        else
            for (int e = 0; e < 4; e++)
                if (d + e < dim) to[e] = (O)x[e];
    };
    constexpr bool share = W > 4;  // a workgroup per item
    constexpr int by = share ? 1 : W, step = share ? W : 1;
    for (int64_t w0 = (int64_t)blockIdx.x * by; w0 < (int64_t)total * chunks; w0 += (int64_t)hidden_blocks * by) {
        const int64_t w = share ? w0 : w0 + wave;
        const int64_t r = w / chunks;
        const int d = (int)(w - r * chunks) * 256 + lane * 4;
        const int i = r < total ? inv[r] : -1;
        f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
        if (i >= 0 && d < dimp) {
#pragma unroll 8
            for (int p = share ? wave : 0; p < parts; p += step)
                x += *reinterpret_cast<const f32x4 *>(part + ((int64_t)p * n + i) * dimp + d);
        }
        if (!share) {
            if (r < total && d < dim) put(r, i, d, x);
            continue;
        }
        red[wave][lane] = x;
        __syncthreads();
        if (wave == 0 && d < dim) {
            for (int k = 1; k < W; k++) x += red[k][lane];
            put(r, i, d, x);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- term weights' small kernels

// The lowest kept row in [f0, f1) whose logit is NaN; f0 if a sum has one in another order only.  Comparisons lose a NaN, and
// to keep it in the tiles' epilogue takes registers that they do not have (step of 32 x 256: 357 -> 569 us), so it is looked
// for where a maximum turned out to be NaN.  A row with a NaN has only NaN logits: a wave finds the text's first (`nan`), and
// the first with an infinity before it (`inf`), whose logits are made again term by term, as those of an infinite term are.  64
// texts of 256 tokens, the last one of each a NaN: 7 ms more (1945 with every row's logits made again).
struct OddRows {
    int inf, nan;
};
template <int HT>
__device__ __forceinline__ OddRows odd_rows(const Source &h, const int *rows, int f0, int f1) {
    using T = typename HVal<HT>::t;
    OddRows o{f1, f1};
    for (int i = f0; i < f1; i++) {
        const T *x = source_row<T>(h, rows[i]);
        bool nan = false, inf = false;
#pragma unroll 4
        for (int d = gs_lane(); d < h.dim; d += 64) {
            const float y = (float)x[d * h.sd];
            nan |= y != y, inf |= fabsf(y) == INFINITY;
        }
        if (__any(nan)) {
            o.nan = i;
            break;
        }
        if (__any(inf)) o.inf = min(o.inf, i);
    }
    return o;
}
template <int HT>
__device__ __forceinline__ int nan_row(const Source &h, const Source &w, float bias, const int *rows, int f0, int f1, int v,
                                       const OddRows &o) {
    using T = typename HVal<HT>::t;
    if (bias != bias) return f0;
    const T *y = source_row<T>(w, v);
    bool inf = false;
#pragma unroll 4
    for (int d = 0; d < h.dim; d++) {
        const float a = (float)y[d * w.sd];
        if (a != a) return f0;
        inf |= fabsf(a) == INFINITY;
    }
    for (int i = inf ? f0 : o.inf; i < o.nan; i++) {
        const T *x = source_row<T>(h, rows[i]);
        float a = 0.f;
        for (int d = 0; d < h.dim && a == a; d++) a = fmaf((float)x[d * h.sd], (float)y[d * w.sd], a);
        if (a + bias != a + bias) return i;
    }
    return o.nan < f1 ? o.nan : f0;
}

// A text's weights from its slots: log(1 + relu(maximum)), and the lowest token that has it (-1 where the weight is 0).  HT:
// the hidden states' type, for the tokens of NaNs.  64 texts of 160 tokens, 30522 terms: 25 MB in 9 us.
template <bool TOK, int HT>
__global__ __launch_bounds__(256) void k_term_weights(const float *best, const int *where, const int *text_first, int block, int vocab,
                                                      const int *rows, int length, float *weights, int *tokens, Source h, Source w,
                                                      const float *bias) {
    const int64_t b = blockIdx.y;
    const int f0 = text_first[b], f1 = text_first[b + 1];
    const int w0 = f0 / block, w1 = (f1 - 1) / block;
    // rows of any length: values of 4 bytes are aligned, groups of four need not be
    typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
    typedef int i4u __attribute__((ext_vector_type(4), aligned(4)));
    for (int v0 = (blockIdx.x * 256 + (int)(threadIdx.x & 192)) * 4; v0 < vocab; v0 += gridDim.x * 1024) {  // whole waves
        const int v = v0 + gs_lane() * 4;
        const bool four = v + 3 < vocab;
        f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
        i4u row = {-1, -1, -1, -1};
        if (f1 > f0) {
            for (int w = w0; w <= w1; w++) {
                const int64_t at = (w + b) * vocab + v;
                f32x4 y = f32x4{0.f, 0.f, 0.f, 0.f};
                i4u wh = row;
                if (four) {
                    y = *reinterpret_cast<const f4u *>(best + at);
                    if (TOK) wh = *reinterpret_cast<const i4u *>(where + at);
                } else {
                    for (int e = 0; v + e < vocab; e++) {
                        y[e] = best[at + e];
                        if (TOK) wh[e] = where[at + e];
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (TOK) row[e] = y[e] > x[e] ? wh[e] : row[e];
                    x[e] = maximum(x[e], y[e], y[e]);
                }
            }
        }
        f4u out;
        i4u tok;
        if (TOK && __any(x[0] != x[0] || x[1] != x[1] || x[2] != x[2] || x[3] != x[3])) {
            const OddRows odd = odd_rows<HT>(h, rows, f0, f1);
#pragma unroll 1
            for (int e = 0; e < 4; e++) {
                const float y = e & 2 ? (e & 1 ? x[3] : x[2]) : (e & 1 ? x[1] : x[0]);
                const int r = y != y ? nan_row<HT>(h, w, bias[v + e], rows, f0, f1, v + e, odd) : -1;
#pragma unroll
                for (int k = 0; k < 4; k++) row[k] = r >= 0 && k == e ? r : row[k];
            }
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            out[e] = log1pf(x[e]);
            if (TOK) tok[e] = row[e] >= 0 ? rows[row[e]] % length : -1;
        }
        const int64_t to = b * vocab + v;
        if (four) {
            *reinterpret_cast<f4u *>(weights + to) = out;
            if (TOK) *reinterpret_cast<i4u *>(tokens + to) = tok;
        } else {
            for (int e = 0; v + e < vocab; e++) {
                weights[to + e] = out[e];
                if (TOK) tokens[to + e] = tok[e];
            }
        }
    }
}

// Term weights of at most 64 rows in one launch, for latency: a workgroup takes 64 terms and all rows where they lie (16-bit,
// 16-byte aligned; rows that the mask leaves out are read as zeros and not looked at), so that there is nothing to list,
// pack or join.  What bounds it is the vocabulary's bytes: 30522 terms of 768 values, 24 rows, 11 us (4.4 TB/s)
// against 27 in four launches.
template <class T, bool TOK>
__global__ __launch_bounds__(256, 2) void k_few_rows(Source h, const uint8_t *mask, Operand W, const void *bias, int bias_type,
                                                     int texts, int length, int vocab, float *weights, int *tokens) {
    constexpr int NS = 4, stage_bytes = 2 * 64 * kStep * 2, loads = 4;
    __shared__ __align__(1024) char smem[NS * stage_bytes];
    const lds_t lds = (lds_t)smem;
    const int lane = gs_lane(), wave = gs_uniform((int)threadIdx.x >> 6);
    const int rows = texts * length, c0 = blockIdx.x * 64;
    const uint64_t kept = __ballot(lane < rows && (!mask || mask[min(lane, rows - 1)] != 0));
    // the rows' pieces: rows 8 wave .. + 7 and 32 further, chunks as in Loader
    int off[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const int row = u * 32 + wave * 8 + lane / 8;
        const int text = row / length;
        off[u] = (kept >> row) & 1
                     ? (int)((text * h.s0 + (row - text * length) * h.s1) * 2) + ((lane % 8) ^ (row & 7)) * 16
                     : 0x7FFFFFF0;
    }
    [[maybe_unused]] const auto hr = gs_rsrc(h.p, (uint32_t)(((texts - 1) * h.s0 + (length - 1) * h.s1 + h.dim) * 2));
    using LW = Loader<64, false, false, 4>;
    Cursor<64, false, false> w;
    w.start(W, c0, vocab, 0, 0, 0);
    [[maybe_unused]] const int w_off = LW::offset(W, wave, lane), w_gap = LW::gap(W);
    const int total = h.dim / kStep;
    auto issue = [&](int st) {
#if defined(__HIP_DEVICE_COMPILE__)
        const lds_t to = lds + (st % NS) * stage_bytes;
#pragma unroll
        for (int u = 0; u < 2; u++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(hr, (__attribute__((address_space(3))) void *)(to + ((wave + u * 4) << 10)), 16,
                                                     off[u], st * kStep * 2, 0, 0);
        LW::issue(w.buffer(W), w_gap, w_off, st * kStep * 2, to + 64 * kStep * 2, wave);
#endif
    };
    const int v = c0 + wave * 16 + (lane & 15);
    float b = 0.f;
    if (bias && v < vocab)
        b = bias_type == GS_H_F32 ? ((const float *)bias)[v]
                                  : bias_type == GS_H_F16 ? (float)((const _Float16 *)bias)[v] : (float)((const __bf16 *)bias)[v];
    Frags<64, false, false, 4> fr;
    Frags<64, false, false, 1> fc;
    fr.init(0, lane);
    fc.init(wave * 16, lane);
    f32x4 acc[4];
#pragma unroll
    for (int i = 0; i < 4; i++) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int st = 0; st < min(NS - 1, total); st++) issue(st);
    for (int it = 0; it < total; it++) {
        if (it + NS - 1 <= total) wait_loads<(NS - 2) * loads>();
        else wait_loads<0>();
        tile_barrier();
        if (it + NS - 1 < total) issue(it + NS - 1);
        const lds_t from = lds + (it % NS) * stage_bytes;
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const s16x8 fb = fc.read(from + 64 * kStep * 2, 0, half);
#pragma unroll
            for (int i = 0; i < 4; i++) acc[i] = T::mfma(fr.read(from, i, half), fb, acc[i]);
        }
    }
    const int q = lane >> 4;
    for (int text = 0; text < texts; text++) {
        const int lo = text * length, hi = lo + length;
        float x = -INFINITY;
        int r = 0x7FFFFFFF;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (16 * i >= hi || 16 * i + 16 <= lo) continue;
            f32x4 y;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int row = 16 * i + 4 * q + e;
                y[e] = row >= lo && row < hi && ((kept >> row) & 1) ? acc[i][e] : -INFINITY;
            }
            EpiTextMax<TOK>::take(y, 16 * i + 4 * q, x, r);
        }
        const auto join = [&](Two<float> x2, Two<int> r2) {
            if (TOK) r = x2.b > x2.a || (x2.b == x2.a && r2.b < r2.a) ? r2.b : r2.a;
            x = maximum(x2.a, x2.b, x2.b);
        };
        join(across<16>(x), TOK ? across<16>(r) : Two<int>{0, 0});
        join(across<32>(x), TOK ? across<32>(r) : Two<int>{0, 0});
        if (TOK && __any(!(x + b > -INFINITY))) {  // no comparison found a NaN's row, see nan_row: the least of these keys does
            int key = 0x7FFFFFFF;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int row = 16 * i + 4 * q + e;
                    const float l = acc[i][e] + b;
                    if (row >= lo && row < hi && ((kept >> row) & 1)) key = min(key, l != l ? row : row + 64);
                }
            const auto least = [&](Two<int> k) { key = min(k.a, k.b); };
            least(across<16>(key));
            least(across<32>(key));
            r = x + b > -INFINITY ? r : key & 63;
        }
        // the bias of a text without a kept row is not looked at either: it may be infinite or NaN
        const bool any = (kept >> lo) & (~0ull >> (64 - length));
        x = any ? maximum(x + b, 0.f, 0.f) : 0.f;
        if (q == 0 && v < vocab) {
            weights[(int64_t)text * vocab + v] = log1pf(x);
            if (TOK) tokens[(int64_t)text * vocab + v] = x > 0.f || x != x ? r - lo : -1;
        }
    }
}

// What k_few8 makes of a block's sums for texts.  The logits but for their column's scale go to LDS, since a text's rows lie in any
// lanes: then a row of lanes takes a text (of four or more), or a fourth of its rows.  (21 texts of 3 tokens of 170 fp32 values, 11762
// terms: 20 us, 44 with maxima taken from registers text by text; 69 of one token of 512, 27652 terms: 27, and 57 as tiles in three
// launches; one of 24, 768, 30522: 11.)
struct EpiFewTerms {
    const void *bias;
    int bias_type, texts, length;
    float *weights;
    static constexpr bool joins = true;
    static constexpr int most_rows = kFewRows;
    __device__ __forceinline__ ColumnScale column(int v, const Weight8 &W) const { return column_scale(v, W, bias, bias_type); }
    __device__ __forceinline__ void block(const i32x4 &sum, int m, int, const Weight8 &, const ColumnScale &col, const float *scales, int, int lane,
                                          float *left) const {
        const int row = 16 * m + 4 * (lane >> 4);
        f32x4 x = __builtin_convertvector(sum, f32x4) * *reinterpret_cast<const f32x4 *>(scales + row);
        if (__builtin_expect(__any(reorders(col.by)), 0)) {
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = in_order(x[e], col);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) left[(row + e) * kFewPitch + (lane & 15)] = x[e];
    }
    // wave `wave` of `waves` that share the values
    __device__ __forceinline__ void finish(const float *left, int v, const Weight8 &W, const ColumnScale &col, const Kept &kept, int lane, int wave,
                                           int waves) const {
        const int q = lane >> 4;
        const bool apart = texts >= 4;  // a text for each row of lanes
        for (int t0 = apart ? wave * 4 : wave; t0 < texts; t0 += apart ? waves * 4 : waves) {
            const int text = apart ? t0 + q : t0, lo = text * length;
            float top = -INFINITY;
            bool any = false;  // the bias of a text without a kept row is not looked at: it may be infinite or NaN
            for (int r = apart ? 0 : q; r < length; r += apart ? 1 : 4) {
                if (text >= texts || !kept(lo + r)) continue;
                const float x = left[(lo + r) * kFewPitch + (lane & 15)];
                top = maximum(top, x, x), any = true;
            }
            if (!apart) {
                const auto join = [&](Two<float> t) { top = maximum(t.a, t.b, t.b); };
                join(across<16>(top));
                join(across<32>(top));
                any = __any(any);
            }
            if (text < texts && v < W.n && (apart || q == 0))
                weights[(int64_t)text * W.n + v] = log1pf(any ? maximum(fmaf(top * fabsf(col.by), kUp, col.bias), 0.f, 0.f) : 0.f);
        }
    }
};

__global__ void k_no_tokens(int64_t n, float *weights, int *tokens) {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        weights[i] = 0.f;
        if (tokens) tokens[i] = -1;
    }
}

// The gradient of the term weights has one entry per (text, term) with a positive weight: g' = g e^-w at the term's token.
// dW adds g' H[token] over texts, dH g' W[term] over a token's terms; for dH a text's entries are sorted by token (terms
// ascending within a token), stably and without an atomic that decides an order, so that every sum has one order.
//
// A wave owns a run of kRun terms.  k_entry_counts: entries per (run, token); k_entry_starts: where they go;
// k_entry_place: there they go.  first[text][length + 1]: the first entry of each token.
constexpr int kRun = 256, kTok = 1024;

// For each entry of the lanes' tokens t (`on`): how many lanes before hold the same token, and how many do in all.
__device__ __forceinline__ void same_token(int t, bool on, int bits, int &rank, int &all) {
    uint64_t same = __ballot(on);
    for (int b = 0; b < bits; b++) {
        const bool one = (t >> b) & 1;
        const uint64_t m = __ballot(on && one);
        same &= one ? m : ~m;
    }
    rank = __popcll(same & gs_lanemask_lt());
    all = __popcll(same);
}

// f(v, t, rank, all) for the run's entries whose token lies in [t0, t0 + kTok); v: the term, t: token - t0
template <class F>
__device__ __forceinline__ void each_entry(const int *tokens, int run, int vocab, int length, int t0, F &&f) {
    const int lane = gs_lane(), most = min(kTok, length - t0);
    const int bits = 32 - __clz(max(most - 1, 1));
    int t[kRun / 64];
#pragma unroll
    for (int c = 0; c < kRun / 64; c++) {
        const int v = run * kRun + c * 64 + lane;
        t[c] = v < vocab ? tokens[v] - t0 : -1;
    }
#pragma unroll
    for (int c = 0; c < kRun / 64; c++) {
        const bool on = t[c] >= 0 && t[c] < most;
        int rank, all;
        same_token(t[c], on, bits, rank, all);
        f(run * kRun + c * 64 + lane, t[c], on, rank, all);
    }
}

__global__ __launch_bounds__(256) void k_entry_counts(const int *tokens, int vocab, int length, int runs, uint16_t *counts) {
    __shared__ int count[4][kTok];
    const int64_t b = blockIdx.y;
    const int lane = gs_lane(), wave = threadIdx.x >> 6, run = blockIdx.x * 4 + wave;
    if (run >= runs) return;
    for (int t0 = 0; t0 < length; t0 += kTok) {
        const int most = min(kTok, length - t0);
        for (int t = lane; t < most; t += 64) count[wave][t] = 0;
        gs_wave_sync();
        each_entry(tokens + b * vocab, run, vocab, length, t0, [&](int, int t, bool on, int rank, int all) {
            if (on && rank == 0) count[wave][t] += all;
            gs_wave_sync();
        });
        uint16_t *to = counts + (b * runs + run) * length + t0;
        for (int t = lane; t < most; t += 64) to[t] = (uint16_t)count[wave][t];
        gs_wave_sync();
    }
}

// starts[text][run][token]: the place of the run's first entry of the token.  One workgroup per text; T tokens at a time, the
// runs in 1024 / T slices, so that short texts have the loads of all threads on their way (120 runs, 64
// tokens: 9.7 -> 5.9 us, 256 tokens: 10.2 -> 9.6).
__global__ __launch_bounds__(1024) void k_entry_starts(const uint16_t *counts, int length, int runs, int *starts, int *first) {
    __shared__ int sums[1024], part[16];
    const int64_t b = blockIdx.x;
    const int tid = threadIdx.x, lane = gs_lane(), wave = tid >> 6;
    const int T = length <= 64 ? 64 : length <= 128 ? 128 : length <= 256 ? 256 : length <= 512 ? 512 : 1024;
    const int slices = 1024 / T, waves = T / 64, g = tid / T;
    const int r0 = runs * g / slices, r1 = runs * (g + 1) / slices;
    int base = 0;
    for (int t0 = 0; t0 < length; t0 += T) {
        const int t = t0 + tid % T;
        const uint16_t *from = counts + b * runs * length + t;
        int *to = starts + b * runs * length + t;
        int c = 0;
        // eight loads at a time, also of the last ones
        const auto load = [&](int r, int (&x)[8]) {
#pragma unroll
            for (int u = 0; u < 8; u++) x[u] = from[(int64_t)min(r + u, r1 - 1) * length];
        };
        if (t < length) {
            for (int r = r0; r < r1; r += 8) {
                int x[8];
                load(r, x);
#pragma unroll
                for (int u = 0; u < 8; u++) c += r + u < r1 ? x[u] : 0;
            }
        }
        sums[tid] = c;
        __syncthreads();
        int before = 0, all = 0;  // of the token: in the slices before this one, in all
        for (int k = 0; k < slices; k++) {
            const int x = sums[k * T + tid % T];
            before += k < g ? x : 0;
            all += x;
        }
        const int inc = (int)gs_wave_incl_scan((uint32_t)all);
        if (lane == 63) part[wave] = inc;
        __syncthreads();
        int at = base + inc - all + before;
        for (int w = 0; w < waves; w++) {
            if (w < wave % waves) at += part[w];
            base += part[w];
        }
        if (t < length) {
            if (g == 0) first[b * (length + 1) + t] = at;
            for (int r = r0; r < r1; r += 8) {
                int x[8];
                load(r, x);
#pragma unroll
                for (int u = 0; u < 8; u++) {
                    if (r + u < r1) to[(int64_t)(r + u) * length] = at;
                    at += x[u];
                }
            }
        }
    }
    if (tid == 0) first[b * (length + 1) + length] = base;
}

struct Entry {
    int v, t;
    float g;
};

__global__ __launch_bounds__(256) void k_entry_place(const float *grad, const float *weights, const int *tokens, int vocab,
                                                     int length, int runs, const int *starts, Entry *entries) {
    __shared__ int next[4][kTok];
    const int64_t b = blockIdx.y;
    const int lane = gs_lane(), wave = threadIdx.x >> 6, run = blockIdx.x * 4 + wave;
    if (run >= runs) return;
    for (int t0 = 0; t0 < length; t0 += kTok) {
        const int most = min(kTok, length - t0);
        const int *from = starts + (b * runs + run) * length + t0;
        for (int t = lane; t < most; t += 64) next[wave][t] = from[t];
        gs_wave_sync();
        each_entry(tokens + b * vocab, run, vocab, length, t0, [&](int v, int t, bool on, int rank, int all) {
            const int at = on ? next[wave][t] : 0;
            gs_wave_sync();
            if (on) {
                // d log(1 + x) / dx = 1 / (1 + x) = e^-w
                entries[b * vocab + at + rank] = Entry{v, t0 + t, grad[b * vocab + v] * expf(-weights[b * vocab + v])};
                if (rank == 0) next[wave][t] = at + all;
            }
            gs_wave_sync();
        });
    }
}

// U rows of up to 256 NC values in a wave's registers, all on their way at once: lane l holds values 256 c + 4 l .. + 3.
// Aligned rows (`vec`) are read through a buffer that ends with the row, so that no lane branches: with the word that holds its
// last value, since one that the buffer ends in reads 0 (the rows are 8-byte aligned, so the word is the row's own memory or
// what pads it).
template <int U, int NC, class T>
__device__ __forceinline__ void rows_load(f32x4 (&x)[U][NC], const T *const (&row)[U], int64_t ds, int d0, int dim, bool vec) {
    const int lane = gs_lane();
    if (vec) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const auto r = gs_rsrc(row[u], (uint32_t)round_up(dim * sizeof(T), 4));
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const int off = (d0 + c * 256 + lane * 4) * (int)sizeof(T);
                Four<T> v;
                if constexpr (sizeof(T) == 4) v = __builtin_bit_cast(Four<T>, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
                else v = __builtin_bit_cast(Four<T>, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
                x[u][c] = f32x4{(float)v.v[0], (float)v.v[1], (float)v.v[2], (float)v.v[3]};
            }
        }
    } else {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int c = 0; c < NC; c++) x[u][c] = row4(row[u], ds, d0 + c * 256 + lane * 4, dim, false);
    }
}
template <int NC, class T>
__device__ __forceinline__ void row_store(T *row, const f32x4 (&x)[NC], int d0, int dim) {
    const bool vec = (dim & 3) == 0;
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int d = d0 + c * 256 + gs_lane() * 4;
        if (vec && d < dim) store4(row + d, x[c]);
        else
            for (int e = 0; e < 4; e++)
                if (d + e < dim) row[d + e] = (T)x[c][e];
    }
}

// dH by chunks of a text's entries, one wave each, whatever tokens they belong to: a token whose entries all lie in the
// chunk is written; a share of one goes to part[chunk][1] where its entries begin in the chunk, else to part[chunk][0].
template <int HT, int NC>
__device__ __forceinline__ void entries_hidden(int block, int64_t b, const void *weight, int64_t wr, int64_t wd, int wvec,
                                               const Entry *entries, const int *first, int vocab, int length, int dim, int chunk,
                                               int chunks, float *part, int dimp, typename HVal<HT>::t *out) {
    using T = typename HVal<HT>::t;
    const int c = block * 4 + (threadIdx.x >> 6), lane = gs_lane();
    const int total = first[b * (length + 1) + length];
    const int lo = c * chunk, hi = min(lo + chunk, total);
    if (c >= chunks || lo >= hi) return;
    const Entry *es = entries + b * vocab;
    const int before = lo > 0 ? es[lo - 1].t : -1, after = hi < total ? es[hi].t : -1;
    constexpr int U = 4;
    for (int d0 = 0; d0 < dim; d0 += NC * 256) {
        f32x4 sum[NC];
#pragma unroll
        for (int k = 0; k < NC; k++) sum[k] = f32x4{0.f, 0.f, 0.f, 0.f};
        int cur = -1;
        auto flush = [&](bool ends) {
            const bool begins = cur != before;
            if (begins && ends) row_store<NC>(out + (b * length + cur) * dim, sum, d0, dim);
            else row_store<NC>(part + ((b * chunks + c) * 2 + (begins ? 1 : 0)) * dimp, sum, d0, dimp);
        };
        for (int e0 = lo; e0 < hi; e0 += 64) {
            const int n = min(64, hi - e0);
            const Entry mine = es[min(e0 + lane, hi - 1)];
            for (int u0 = 0; u0 < n; u0 += U) {
                f32x4 x[U][NC];
                const T *row[U];
                float g[U];
                int t[U];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int l = min(u0 + u, n - 1);
                    const int v = __builtin_amdgcn_readlane(mine.v, l);
                    t[u] = __builtin_amdgcn_readlane(mine.t, l);
                    g[u] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, mine.g), l));
                    row[u] = (const T *)weight + v * wr;
                }
                rows_load<U, NC, T>(x, row, wd, d0, dim, wvec);
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (u0 + u >= n) break;
                    if (t[u] != cur) {
                        if (cur >= 0) flush(true);
                        cur = t[u];
#pragma unroll
                        for (int k = 0; k < NC; k++) sum[k] = f32x4{0.f, 0.f, 0.f, 0.f};
                    }
#pragma unroll
                    for (int k = 0; k < NC; k++) sum[k] += g[u] * x[u][k];
                }
            }
        }
        flush(cur != after);
    }
}

// What entries_hidden left open: zeros for tokens without entries, sums of the shares of those in several chunks.
template <int HT>
__global__ __launch_bounds__(256) void k_entries_join(const int *first, int64_t rows, int length, int dim, int chunk, int chunks,
                                                      const float *part, int dimp, typename HVal<HT>::t *out) {
    const int lane = gs_lane();
    const bool vec = (dim & 3) == 0;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += (int64_t)gridDim.x * 4) {
        const int64_t b = r / length, t = r % length;
        const int lo = first[b * (length + 1) + t], hi = first[b * (length + 1) + t + 1];
        const int c0 = lo / chunk, c1 = (hi - 1) / chunk;
        if (hi > lo && c0 == c1) continue;
        for (int d = lane * 4; d < dim; d += 256) {
            f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
            if (hi > lo) {
                const float *p = part + (b * chunks + c0) * 2 * dimp + d;
                x = *reinterpret_cast<const f32x4 *>(p + dimp);
#pragma unroll 4
                for (int c = c0 + 1; c <= c1; c++) x += *reinterpret_cast<const f32x4 *>(p + (int64_t)(c - c0) * 2 * dimp);
            }
            auto *to = out + r * dim + d;
            if (vec) store4(to, x);
            else
                for (int e = 0; e < 4; e++)
                    if (d + e < dim) to[e] = (typename HVal<HT>::t)x[e];
        }
    }
}

// dW[v] = sum over texts of g' H[text, token], db[v] = sum of g', texts in order: a workgroup per 16 terms, a wave per 4 of
// them, four rows of hidden states on their way at a time.
template <int HT, int NC>
__device__ __forceinline__ void entries_weight(int block, const Source &h, const float *grad, const float *weights, const int *tokens,
                                               int texts, int vocab, typename HVal<HT>::t *dw, void *db, int db_type) {
    using T = typename HVal<HT>::t;
    __shared__ float sg[64][17];
    __shared__ int st[64][17];
    const int lane = gs_lane(), wave = threadIdx.x >> 6, tid = threadIdx.x;
    const int v0 = block * 16;
    constexpr int U = 4;
    for (int d0 = 0; d0 < h.dim; d0 += NC * 256) {
        f32x4 sum[4][NC];
        float bs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int c = 0; c < NC; c++) sum[u][c] = f32x4{0.f, 0.f, 0.f, 0.f};
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
                const int t = st[lane][wave * 4 + u];
                const float g = sg[lane][wave * 4 + u];
                uint64_t left = __ballot(t >= 0);
                while (left) {
                    f32x4 x[U][NC];
                    const T *row[U];
                    float gl[U];
                    bool live[U];
                    int l = 0;
#pragma unroll
                    for (int k = 0; k < U; k++) {  // past the last entry: its row again, not used
                        const bool on = left != 0;
                        l = on ? __ffsll((unsigned long long)left) - 1 : l;
                        left &= left - 1;
                        const int tl = __builtin_amdgcn_readlane(t, l);
                        gl[k] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, g), l));
                        live[k] = on;
                        row[k] = (const T *)h.p + (int64_t)(b0 + l) * h.s0 + (int64_t)tl * h.s1;
                    }
                    rows_load<U, NC, T>(x, row, h.sd, d0, h.dim, h.vec);
#pragma unroll
                    for (int k = 0; k < U; k++) {
                        if (!live[k]) break;
                        bs[u] += gl[k];
#pragma unroll
                        for (int c = 0; c < NC; c++) sum[u][c] += gl[k] * x[k][c];
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int v = v0 + wave * 4 + u;
            if (v >= vocab) continue;
            if (dw) row_store<NC>(dw + (int64_t)v * h.dim, sum[u], d0, h.dim);
            if (db && d0 == 0 && lane == 0) {
                if (db_type == GS_H_F32) ((float *)db)[v] = bs[u];
                else if (db_type == GS_H_F16) ((_Float16 *)db)[v] = (_Float16)bs[u];
                else ((__bf16 *)db)[v] = (__bf16)bs[u];
            }
        }
    }
}

// Both in one launch: workgroups [0, weight_blocks) take terms, the others chunks of the texts' entries.  Either gathers a row
// of 16-bit values per entry, mostly from the L2: 0.24 M entries of 384 values 48 us, a write of 23 MB among it.
template <int HT, int NC>
__global__ __launch_bounds__(256) void k_entry_sums(Source h, Source w, const float *grad, const float *weights, const int *tokens,
                                                    const Entry *entries, const int *first, int texts, int vocab, int chunk,
                                                    int chunks, float *part, int dimp, typename HVal<HT>::t *dh,
                                                    typename HVal<HT>::t *dw, void *db, int db_type, int weight_blocks) {
    const int block = (int)blockIdx.x - weight_blocks;
    if (block < 0) {
        entries_weight<HT, NC>((int)blockIdx.x, h, grad, weights, tokens, texts, vocab, dw, db, db_type);
    } else {
        const int per = (chunks + 3) / 4;
        entries_hidden<HT, NC>(block % per, block / per, w.p, w.s1, w.sd, w.vec, entries, first, vocab, h.length, h.dim, chunk,
                               chunks, part, dimp, dh);
    }
}

// ---------------------------------------------------------------- host

// Tiles.  A tile's operands cross LDS once per wave that shares them, so larger ones feed the matrix units better; but a
// tile needs work for every CU, and few rows leave the vocabulary's bytes as what takes the time.  The rule looks at the rows
// of a call, kept or not, since the host does not know how many are, and not at the terms: it was measured at one number of
// them.  30522 terms of 768 bf16 values, microseconds of the product alone:
//   rows    64 x 64   256 x 128   256 x 256
//     45       11.4        13.0        18.5
//    128       13.5        13.5        18.7
//    200       22.9        14.8        19.2
//    320       27.3        23.5        20.3
//   1250       90.5        57.2        53.7
// fp32, whole gradient of a loss with 384 values: 77 rows 138 in 64 x 64, 128 in 256 x 128; 256 rows 239, 190.
// k-major operands (dH, dW) do better with waves of 64 x 128 than of 128 x 64 (dW 880 -> 915 TFLOP/s).
template <class T, int NP, bool RK, bool CK, bool CB = false>
using Small = Tile<T, NP, 64, 64, 2, 2, 4, 2, RK, CK, CB>;
template <class T, int NP, bool RK, bool CK, bool CB = false>
using Wide = Tile<T, NP, 256, 128, 4, 2, 3, 2, RK, CK, CB>;
template <class T, int NP, bool RK, bool CK, bool CB = false>  // tokens as rows
using Flat = Tile<T, NP, 128, 256, 2, 4, 3, 2, RK, CK, CB>;
template <class T, int NP, bool RK, bool CK, bool CB = false>
using Large = Tile<T, NP, 256, 256, 2, 4, 2, 2, RK, CK, CB>;
template <class T, int NP, bool RK, bool CK, bool CB = false>
using LargeK = Tile<T, NP, 256, 256, 4, 2, 2, 2, RK, CK, CB>;

constexpr int kSmallRows = 64, kWideRows = 256;

enum TileClass { kSmall, kWide, kLarge };
TileClass class_of(int64_t rows) { return rows <= kSmallRows ? kSmall : rows <= kWideRows ? kWide : kLarge; }
// tokens of a tile
int token_edge(TileClass c) { return c == kSmall ? 64 : c == kWide ? 128 : 256; }
// terms of a tile of the losses, terms of a wave of it, and waves along its tokens
int term_edge(TileClass c) { return c == kSmall ? 64 : 256; }
int term_block(TileClass c) { return c == kSmall ? 32 : c == kWide ? 64 : 128; }
int token_waves(TileClass c) { return c == kLarge ? 4 : 2; }
// tokens of a wave where they are the rows
int token_block(TileClass c) { return token_edge(c) / 2; }

// CALL(operand type, planes) for a head's type
#define GSV_BY_TYPE(type, CALL)              \
    switch (type) {                          \
        case GS_H_F32: CALL(Bf16, 3); break; \
        case GS_H_F16: CALL(F16, 1); break;  \
        default: CALL(Bf16, 1); break;       \
    }
// CALL(value type) for a type of values
#define GSV_BY_VALUE(type, CALL)             \
    switch (type) {                          \
        case GS_H_F32: CALL(float); break;   \
        case GS_H_F16: CALL(_Float16); break; \
        default: CALL(__bf16); break;        \
    }

bool vec_ok(const void *p, int type, int64_t s0, int64_t s1, int64_t sd) {
    return sd == 1 && s0 % 4 == 0 && s1 % 4 == 0 && (uintptr_t)p % (type == GS_H_F32 ? 16 : 8) == 0;
}

int check_head(const gs_vocab_head *h) {
    GS_REQUIRE(h, "head is NULL");
    GS_REQUIRE(known(h->type), "unknown hidden type %d", h->type);
    GS_REQUIRE(known(h->bias_type), "unknown bias type %d", h->bias_type);
    GS_REQUIRE(h->texts >= 0 && h->length >= 0, "negative texts or length");
    GS_REQUIRE((int64_t)h->texts * h->length <= (1 << 28), "%lld rows exceed 2^28", (long long)h->texts * h->length);
    GS_REQUIRE(h->dim >= 1 && h->dim <= 32768, "dim=%d outside [1, 32768]", h->dim);
    GS_REQUIRE(h->vocab >= 1 && h->vocab <= (1 << 20), "vocab=%d outside [1, 2^20]", h->vocab);
    return GS_OK;
}

// Of term weights, which have a grid row per text
int check_texts(const gs_vocab_head *h) {
    if (int rc = check_head(h)) return rc;
    GS_REQUIRE(h->texts <= 65535, "texts=%d exceed 65535", h->texts);
    return GS_OK;
}

// What a call that launches reads of a head
int check_data(const gs_vocab_head *h) {
    GS_REQUIRE(h->weight_d && (h->hidden_d || (int64_t)h->texts * h->length == 0), "NULL hidden states or weight");
    return GS_OK;
}

struct Layout {
    int rows, dimp, planes, vocabp;
    bool w_direct;
    TileClass cls;
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
    l.cls = class_of(l.rows);
    return l;
}

// What every call makes first.
struct Common {
    int *n, *rows, *inv, *seg, *text_first;
    float *bias;
    uint16_t *hidden, *weight;
};

void take_common(gs_arena &a, const Layout &l, const gs_vocab_head *h, bool texts, Common *s) {
    s->n = a.take<int>(64);
    s->rows = a.take<int>(l.rows);
    s->inv = texts ? nullptr : a.take<int>(l.rows);
    s->seg = texts ? a.take<int>(l.rows + kRowPad) : nullptr;
    s->text_first = texts ? a.take<int>(h->texts + 1) : nullptr;
    s->bias = a.take<float>(l.vocabp);
    s->hidden = a.take<uint16_t>((size_t)l.rows * l.planes * l.dimp);
}

// The last of a buffer: whether there is a copy moves nothing else.  A loss and its gradient may be given the weight at
// different places (autograd's hooks on saved tensors bring it back where they like); a gradient that can read it where it
// is does, whether or not the loss copied it.
void take_weight(gs_arena &a, const Layout &l, const gs_vocab_head *h, Common *s) {
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

Operand hidden_operand(const Layout &l, const Common &s) {
    return Operand{s.hidden, (int64_t)l.planes * l.dimp, l.dimp, (int64_t)l.planes * l.dimp};
}
Operand weight_operand(const Layout &l, const Common &s, const gs_vocab_head *h) {
    if (l.w_direct) return Operand{(const uint16_t *)h->weight_d, h->weight_row_stride, 0, l.dimp};
    return Operand{s.weight, (int64_t)l.planes * l.dimp, l.dimp, (int64_t)l.planes * l.dimp};
}

// Kept rows, bias, cleared memory; then hidden states, (where needed) vocabulary rows and targets in the product's form.
int prepare(const gs_vocab_head *h, const Layout &l, const Keep &keep, const Common &c, float *zero, int64_t zeros,
            const TargetRows &targets, const TeacherRows &teacher, hipStream_t s) {
    hipLaunchKernelGGL(k_setup, dim3(1 + gs_blocks(l.vocabp + zeros / 4, 1024, 1024)), dim3(1024), 0, s, keep,
                       h->length > 0 ? h->length : 1, c.rows, c.inv, c.seg, c.text_first, c.n, h->bias_d, h->bias_type, h->vocab,
                       l.vocabp, c.bias, zero, zeros);
    GS_CHECK_LAUNCH();
    const int w_rows = l.w_direct ? 0 : h->vocab;
    if (l.rows + w_rows == 0) return GS_OK;
    const dim3 g(gs_blocks((targets.targets || teacher.ids ? 2 : 1) * (int64_t)l.rows + w_rows, 4, 8192));
    const Source hs = hidden_source(h), ws = weight_source(h);
#define GSV_PACK(HT, NP)                                                                                                     \
    hipLaunchKernelGGL((k_pack<HT, NP>), g, dim3(256), 0, s, hs, c.rows, c.n, c.hidden, ws, w_rows, c.weight, l.dimp, targets, \
                       teacher)
    if (h->type == GS_H_F32) GSV_PACK(GS_H_F32, 3);
    else if (h->type == GS_H_F16) GSV_PACK(GS_H_F16, 1);
    else GSV_PACK(GS_H_BF16, 1);
#undef GSV_PACK
    GS_CHECK_LAUNCH();
    return GS_OK;
}

// ---------------------------------------------------------------- losses

struct LossPlan {
    Layout l;
    int top;
    int piece, pieces;   // terms per piece (a multiple of kRowPad)
    int blocks;          // blocks of softmax sums
    int most;            // parts of dH
    int64_t part_rows;   // rows of all of dH's parts
    int64_t sum_rows;    // rows of the bias's sums
    bool f16;
};

LossPlan loss_plan(const gs_vocab_head *h, const gs_vocab_targets *t, int cus) {
    LossPlan p;
    p.l = layout_of(h);
    p.f16 = h->type == GS_H_F16;
    p.top = t->teacher_ids_d ? t->top : 1;
    const int64_t per = (int64_t)(p.l.rows > 0 ? p.l.rows : 1) * p.l.planes * 2;
    int64_t most = (int64_t)kPieceBytes / per / kRowPad * kRowPad;
    if (most < kRowPad) most = kRowPad;
    p.pieces = (int)((p.l.vocabp + most - 1) / most);
    p.piece = (int)round_up((p.l.vocabp + p.pieces - 1) / p.pieces, kRowPad);
    p.pieces = (p.l.vocabp + p.piece - 1) / p.piece;
    p.blocks = (h->vocab + term_edge(p.l.cls) - 1) / term_edge(p.l.cls) * (term_edge(p.l.cls) / term_block(p.l.cls));
    p.most = p.piece / kStep / 3 < 128 ? p.piece / kStep / 3 : 128;
    if (p.most < 1) p.most = 1;
    // parts_of: parts that even out hold at most a piece's terms and the rows, parts that fill at most a tile's rows for
    // each workgroup that runs at a time
    const int tr = (h->dim + term_edge(p.l.cls) - 1) / term_edge(p.l.cls);
    const int64_t even = (int64_t)p.piece + p.l.rows, fill = (int64_t)2 * cus * token_edge(p.l.cls) / tr + p.l.rows;
    const int64_t by_most = (int64_t)p.most * p.l.rows;
    p.part_rows = even > fill ? even : fill;
    if (p.part_rows > by_most) p.part_rows = by_most;
    p.sum_rows = (int64_t)(p.l.rows + token_edge(p.l.cls) - 1) / token_edge(p.l.cls) * token_waves(p.l.cls);
    return p;
}

struct LossSaved {
    Common c;
    float *lse2, *loss;
    int *ids;          // kept rows' entries
    float *share;
    uint16_t *first;
};

void take_loss_saved(gs_arena &a, const LossPlan &p, const gs_vocab_head *h, const gs_vocab_targets *t, LossSaved *s) {
    const bool teacher = t->teacher_ids_d != nullptr;
    take_common(a, p.l, h, false, &s->c);
    s->lse2 = a.take<float>(p.l.rows);
    s->loss = a.take<float>(p.l.rows);
    s->ids = a.take<int>((size_t)p.l.rows * p.top);
    s->share = teacher ? a.take<float>((size_t)p.l.rows * p.top) : nullptr;
    s->first = teacher ? a.take<uint16_t>((size_t)(p.l.vocabp / term_block(p.l.cls) + 1) * p.l.rows) : nullptr;
    take_weight(a, p.l, h, &s->c);
}

struct LossScratch {
    uint8_t *keep;
    int *ids;          // source rows' entries of a teacher
    float *share, *ent;
    float *target;
    float2 *part;
    float *dots;
};
void take_loss_scratch(gs_arena &a, const LossPlan &p, const gs_vocab_targets *t, LossScratch *s) {
    const bool teacher = t->teacher_ids_d != nullptr;
    const size_t rows = p.l.rows, sums = (size_t)p.blocks * rows;
    s->keep = teacher ? a.take<uint8_t>(rows) : nullptr;
    s->ids = teacher ? a.take<int>(rows * p.top) : nullptr;
    s->share = teacher ? a.take<float>(rows * p.top) : nullptr;
    s->ent = teacher ? a.take<float>(rows) : nullptr;
    s->target = teacher ? nullptr : a.take<float>(rows);
    s->part = a.take<float2>(sums);
    s->dots = teacher ? a.take<float>(sums) : nullptr;
}

struct GradScratch {
    RowFactors rows;
    float *sums, *part;
    int *parts;
    uint16_t *dl;
};
void take_grad_scratch(gs_arena &a, const LossPlan &p, GradScratch *s) {
    s->rows.factor = a.take<float>(p.l.rows);
    s->rows.scale = a.take<float>(64);
    s->rows.own = p.f16 ? a.take<float>(p.l.rows) : nullptr;
    s->rows.undo = p.f16 ? a.take<float>(p.l.rows) : nullptr;
    s->parts = a.take<int>(64);
    s->rows.n_own = s->parts + 1;
    s->sums = a.take<float>((size_t)p.sum_rows * p.l.vocabp);
    s->part = a.take<float>((size_t)p.part_rows * p.l.dimp);
    s->dl = a.take<uint16_t>((size_t)round_up(p.l.rows, kBlock) * p.l.planes * p.piece);
}

int check_targets(const gs_vocab_head *h, const gs_vocab_targets *t) {
    GS_REQUIRE(t, "targets are NULL");
    GS_REQUIRE((t->targets_d != nullptr) != (t->teacher_ids_d != nullptr) || (int64_t)h->texts * h->length == 0,
               "targets or a teacher's ids, not both or neither");
    if (t->teacher_ids_d) {
        GS_REQUIRE(t->teacher_logits_d, "teacher ids without logits");
        GS_REQUIRE(t->top >= 1 && t->top <= kMaxTop, "top=%d outside [1, %d]", t->top, kMaxTop);
        GS_REQUIRE(known(t->teacher_type), "unknown teacher type %d", t->teacher_type);
        GS_REQUIRE(t->temperature > 0.f && t->temperature < INFINITY, "temperature=%g must be positive and finite",
                   (double)t->temperature);
    }
    return GS_OK;
}

float tau_of(const gs_vocab_targets *t) { return t->teacher_ids_d ? t->temperature : 1.f; }

Entries entries_of(const LossPlan &p, const LossSaved &s) { return Entries{s.ids, s.share, s.first, p.l.rows, p.top}; }

template <class T, int NP>
int run_sums(const gs_vocab_head *h, const LossPlan &p, const LossSaved &s, const LossScratch &x, float scale, int cus,
             hipStream_t st) {
    const Dims d{h->vocab, p.l.rows, p.l.dimp, s.c.n, 0, 1, 0};
    const Operand w = weight_operand(p.l, s.c, h), hid = hidden_operand(p.l, s.c);
#define GSV_SUMS(TL)                                                                                                     \
    return s.share ? launch_product<TL<T, NP, false, false>>(                                                            \
                         w, hid, d, EpiSums<true>{s.c.bias, scale, x.part, x.dots, p.l.rows, entries_of(p, s)}, cus, st)  \
                   : launch_product<TL<T, NP, false, false>>(                                                            \
                         w, hid, d, EpiSums<false>{s.c.bias, scale, x.part, x.dots, p.l.rows, entries_of(p, s)}, cus, st)
    switch (p.l.cls) {
        case kSmall: GSV_SUMS(Small);
        case kWide: GSV_SUMS(Wide);
        default: GSV_SUMS(Large);
    }
#undef GSV_SUMS
}

template <class T, int NP, class O>
int run_grad(const gs_vocab_head *h, const LossPlan &p, const LossSaved &s, const GradScratch &g, float scale, const Upstream &up,
             const float *factor, const int *n, const int *n_dh, float power, bool want_dh, bool want_db, void *dw_d, int cus, hipStream_t st) {
    using S = typename T::store_t;
    const Operand w = weight_operand(p.l, s.c, h), hid = hidden_operand(p.l, s.c);
    const int64_t row = (int64_t)p.piece * kBlock;  // values of a row of blocks
    const Operand dl{g.dl, NP * row, row, NP * row};
    for (int c = 0; c < p.pieces; c++) {
        const int v0 = c * p.piece, nv = min(p.piece, h->vocab - v0);
        if (nv <= 0) break;
        Operand wp = w;
        wp.p += (int64_t)v0 * w.stride;
        const EpiHiddenPart eh{g.part, p.l.dimp, c > 0};
        const EpiWeightGrad<O> ew{(O *)dw_d + (int64_t)v0 * h->dim, up, h->dim, h->dim % 4 == 0};
        const Dims de{nv, p.l.rows, p.l.dimp, n, 0, 1, 0};
        const Dims dh{want_dh ? h->dim : 0, p.l.rows, nv, n_dh, 0, 1, 0};
        const Dims dw{dw_d ? h->dim : 0, nv, p.l.rows, n, 0, 0, 1}, none{0, 0, 0, n, 0, 0, 0};
        int rc = GS_OK;
#define GSV_EPI(SHARES) \
    EpiLogitGrad<S, SHARES> { s.c.bias, scale, s.lse2, factor, power, power == 2048.f ? 11.f : 0.f, entries_of(p, s), v0, g.dl, dl.stride, dl.plane, want_db ? g.sums : nullptr, p.l.vocabp }
#define GSV_GRAD(TL)                                                                              \
    rc = s.share ? launch_product<TL<T, NP, false, false>>(wp, hid, de, GSV_EPI(true), cus, st)   \
                 : launch_product<TL<T, NP, false, false>>(wp, hid, de, GSV_EPI(false), cus, st)
        switch (p.l.cls) {
            case kSmall: GSV_GRAD(Small); break;
            case kWide: GSV_GRAD(Wide); break;
            default: GSV_GRAD(Large); break;
        }
#undef GSV_GRAD
#undef GSV_EPI
        if (rc) return rc;
        if (!want_dh && !dw_d) continue;
#define GSV_PAIR(TL, DW)                                                                                              \
    rc = launch_pair<TL<T, NP, true, false, true>, TL<T, NP, true, true, true>>(wp, dl, dh, eh, hid, dl, DW, ew, p.piece, p.most, \
                                                                    g.parts, cus, st)
        switch (p.l.cls) {
            case kSmall:
                // few rows: dW is its output's bytes, which larger tiles write faster
                GSV_PAIR(Small, none);
                if (!rc) rc = launch_product<Wide<T, NP, true, true, true>>(hid, dl, dw, ew, cus, st);
                break;
            case kWide: GSV_PAIR(Wide, dw); break;
            default: GSV_PAIR(LargeK, dw); break;
        }
#undef GSV_PAIR
        if (rc) return rc;
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
    int cus = 0;
    if (int rc = cu_count(&cus)) return rc;
    const LossPlan p = loss_plan(h, t, cus);
    LossSaved s;
    LossScratch x;
    GradScratch g;
    gs_arena a{nullptr, 0, 0}, b{nullptr, 0, 0}, c{nullptr, 0, 0};
    take_loss_saved(a, p, h, t, &s);
    take_loss_scratch(b, p, t, &x);
    take_grad_scratch(c, p, &g);
    *saved_bytes = a.used, *scratch_bytes = b.used, *grad_bytes = c.used;
    return GS_OK;
}

extern "C" int gs_vocab_loss(const gs_vocab_head *h, const gs_vocab_targets *t, int32_t reduction, float *loss_d, void *saved_d,
                             size_t saved_bytes, void *scratch_d, size_t scratch_bytes, void *stream) {
    if (int rc = check_head(h)) return rc;
    if (int rc = check_targets(h, t)) return rc;
    GS_REQUIRE(reduction >= GS_REDUCE_NONE && reduction <= GS_REDUCE_SUM, "unknown reduction %d", reduction);
    GS_REQUIRE(saved_d && (loss_d || (reduction == GS_REDUCE_NONE && (int64_t)h->texts * h->length == 0)), "NULL loss or workspace");
    int cus = 0;
    if (int rc = cu_count(&cus)) return rc;
    const LossPlan p = loss_plan(h, t, cus);
    LossSaved sv;
    LossScratch x;
    gs_arena a{(char *)saved_d, 0, saved_bytes}, b{(char *)scratch_d, 0, scratch_bytes};
    take_loss_saved(a, p, h, t, &sv);
    take_loss_scratch(b, p, t, &x);
    GS_REQUIRE(scratch_d || b.used == 0, "NULL workspace");
    if (!a.ok() || !b.ok()) {
        gs_set_error("vocab_loss workspace too small: need %zu + %zu bytes, got %zu + %zu", a.used, b.used, saved_bytes,
                     scratch_bytes);
        return GS_ENOSPC;
    }
    if (int rc = check_data(h)) return rc;
    const hipStream_t s = gs_stream(stream);
    const int rows = p.l.rows;
    const float tau = tau_of(t);
    const bool teacher = t->teacher_ids_d != nullptr;
    if (teacher && rows > 0) {
        const int th = t->top <= 64 ? 64 : t->top <= 128 ? 128 : 256;
        hipLaunchKernelGGL(k_teacher, dim3(rows), dim3(th), 0, s, t->teacher_ids_d, t->teacher_logits_d, t->teacher_type, t->top,
                           h->vocab, 1.f / tau, x.ids, x.share, x.ent, x.keep);
        GS_CHECK_LAUNCH();
    }
    const Keep keep{x.keep, teacher ? nullptr : t->targets_d, t->ignore_index, h->vocab, rows};
    const TargetRows targets{teacher ? nullptr : t->targets_d, sv.c.bias, sv.ids, x.target};
    const TeacherRows entries{teacher ? x.ids : nullptr, x.share, p.top, p.l.vocabp / term_block(p.l.cls), term_block(p.l.cls), rows, sv.ids, sv.share, sv.first};
    if (int rc = prepare(h, p.l, keep, sv.c, loss_d, reduction == GS_REDUCE_NONE ? rows : 0, targets, entries, s)) return rc;
    if (rows > 0) {
        int rc = GS_OK;
#define GSV_SUMS(T, NP) rc = run_sums<T, NP>(h, p, sv, x, kLog2e / tau, cus, s)
        GSV_BY_TYPE(h->type, GSV_SUMS)
#undef GSV_SUMS
        if (rc) return rc;
#define GSV_RL(X)                                                                                                          \
    hipLaunchKernelGGL(k_row_loss<X>, dim3(gs_blocks(rows, X, 4096)), dim3(256), 0, s, x.part, x.dots, (int64_t)rows, p.blocks, \
                       sv.c.rows, sv.c.n, x.target, x.ent, tau, sv.lse2, sv.loss, reduction == GS_REDUCE_NONE ? loss_d : nullptr)
        if (rows <= 1024) GSV_RL(4);
        else GSV_RL(16);
#undef GSV_RL
        GS_CHECK_LAUNCH();
    }
    if (reduction != GS_REDUCE_NONE) {
        hipLaunchKernelGGL(k_loss_sum, dim3(1), dim3(1024), 0, s, sv.loss, sv.c.n, reduction == GS_REDUCE_MEAN, loss_d);
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
    GS_REQUIRE(saved_d && scratch_d && (grad_d || (reduction == GS_REDUCE_NONE && (int64_t)h->texts * h->length == 0)), "NULL gradient or workspace");
    int cus = 0;
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
    GS_REQUIRE(h->weight_d, "NULL weight");
    const hipStream_t s = gs_stream(stream);
    const int rows = p.l.rows;
    const float tau = tau_of(t);
    const bool per_row = reduction == GS_REDUCE_NONE, f16 = p.f16;
    if (per_row) {
        hipLaunchKernelGGL(k_row_factor, dim3(1), dim3(1024), 0, s, grad_d, sv.c.rows, sv.c.n, tau, g.rows);
        GS_CHECK_LAUNCH();
    }
    const float power = f16 && !per_row ? 2048.f : 1.f;
    const Upstream up{grad_d, sv.c.n, reduction == GS_REDUCE_MEAN, tau / power, per_row ? g.rows.scale : nullptr};
    int rc = GS_OK;
    // without a kept row no launch has a tile but dW's, which writes its zeros
#define GSV_RUN(T, NP, O, FACTOR, N, N_DH, DB, DW) \
    rc = run_grad<T, NP, O>(h, p, sv, g, kLog2e / tau, up, FACTOR, N, N_DH, power, dhidden_d, DB, DW, cus, s)
    const bool own = per_row && f16 && dhidden_d;
    const float *factor = per_row ? g.rows.factor : nullptr;
    if (h->type == GS_H_F32) GSV_RUN(Bf16, 3, float, factor, sv.c.n, sv.c.n, dbias_d, dweight_d);
    else if (f16) GSV_RUN(F16, 1, _Float16, factor, sv.c.n, own ? g.rows.n_own + 1 : sv.c.n, dbias_d, dweight_d);
    else GSV_RUN(Bf16, 1, __bf16, factor, sv.c.n, sv.c.n, dbias_d, dweight_d);
    if (own && !rc) GSV_RUN(F16, 1, _Float16, g.rows.own, g.rows.n_own, g.rows.n_own, false, nullptr);
#undef GSV_RUN
    if (rc) return rc;
    const int64_t items = dhidden_d ? (int64_t)rows * ((h->dim + 255) / 256) : 0;
    const bool few = items <= 1024;
    const int hidden_blocks = items ? (int)gs_blocks(items, few ? 1 : 4, 8192) : 0;
    const int bias_blocks = dbias_d ? (h->vocab + 31) / 32 : 0;
    if (hidden_blocks + bias_blocks == 0) return GS_OK;
    const BiasSums bias{g.sums, p.l.vocabp, token_edge(p.l.cls), token_waves(p.l.cls), h->vocab, h->bias_type, dbias_d};
#define GSV_FG(O, W)                                                                                                       \
    hipLaunchKernelGGL((k_finish_grad<O, W>), dim3(hidden_blocks + bias_blocks), dim3(64 * W), 0, s, g.part, sv.c.inv, sv.c.n, \
                       g.parts, rows, h->dim, p.l.dimp, up, own ? g.rows.undo : nullptr, (O *)dhidden_d, hidden_blocks, bias)
#define GSV_FINISH(O)               \
    if (few) GSV_FG(O, 16);         \
    else GSV_FG(O, 4)
    GSV_BY_VALUE(h->type, GSV_FINISH)
#undef GSV_FINISH
#undef GSV_FG
    GS_CHECK_LAUNCH();
    return GS_OK;
}

// ---------------------------------------------------------------- term weights

namespace gsv {

// Slots of the maxima: a block of a wave's rows and a text each make one more.
size_t text_slots(const gs_vocab_head *h, const Layout &l) {
    const int block = token_block(l.cls);
    return (size_t)(l.rows + block - 1) / block + h->texts;
}

struct EntryPlan {
    int runs, chunk, chunks, dimp;
    Entry *entries;
    int *first, *starts;
    uint16_t *counts;
    float *part;
};
// Chunks of 64 entries fill the GPU on small batches; larger ones take fewer open ends (two rows of fp32 a chunk).
void take_entries(gs_arena &a, const gs_vocab_head *h, EntryPlan *p) {
    const size_t n = (size_t)h->texts * h->vocab, rows = (size_t)h->texts * h->length;
    p->runs = (h->vocab + kRun - 1) / kRun;
    p->chunk = n <= (size_t)4 << 20 ? 64 : 256;
    p->chunks = (h->vocab + p->chunk - 1) / p->chunk;
    p->dimp = (int)round_up(h->dim, 4);
    p->entries = a.take<Entry>(n);
    p->first = a.take<int>(rows + h->texts);
    p->starts = a.take<int>(rows * p->runs);
    p->counts = a.take<uint16_t>(rows * p->runs);
    p->part = a.take<float>((size_t)h->texts * p->chunks * 2 * p->dimp);
}

// Whether k_few_rows may read hidden states and vocabulary where they are.
bool few_rows_ok(const gs_vocab_head *h, const Layout &l) {
    const int64_t span = (int64_t)(h->texts - 1) * h->hidden_text_stride + (int64_t)(h->length - 1) * h->hidden_row_stride + h->dim;
    return l.w_direct && h->hidden_dim_stride == 1 && h->hidden_text_stride % 8 == 0 && h->hidden_row_stride % 8 == 0 &&
           h->hidden_text_stride >= 0 && h->hidden_row_stride >= 0 && (uintptr_t)h->hidden_d % 16 == 0 && span < (1 << 29);
}

// f(NC) for the registers a row of `dim` values takes, 256 a piece
#define GSV_BY_CHUNKS(dim, CALL)              \
    switch (((dim) + 255) / 256) {            \
        case 1: CALL(1); break;               \
        case 2: CALL(2); break;               \
        case 3: CALL(3); break;               \
        default: CALL(4); break;              \
    }

template <int HT>
int run_entries(const gs_vocab_head *h, const float *grad_d, const float *weights_d, const int32_t *tokens_d, void *dhidden_d,
                void *dweight_d, void *dbias_d, const EntryPlan &p, hipStream_t s) {
    using T = typename HVal<HT>::t;
    const int64_t rows = (int64_t)h->texts * h->length;
    const Source ws = weight_source(h), hs = hidden_source(h);
    if (dhidden_d && rows > 0) {
        const dim3 g((p.runs + 3) / 4, h->texts);
        hipLaunchKernelGGL(k_entry_counts, g, dim3(256), 0, s, tokens_d, h->vocab, h->length, p.runs, p.counts);
        GS_CHECK_LAUNCH();
        hipLaunchKernelGGL(k_entry_starts, dim3(h->texts), dim3(1024), 0, s, p.counts, h->length, p.runs, p.starts, p.first);
        GS_CHECK_LAUNCH();
        hipLaunchKernelGGL(k_entry_place, g, dim3(256), 0, s, grad_d, weights_d, tokens_d, h->vocab, h->length, p.runs, p.starts,
                           p.entries);
        GS_CHECK_LAUNCH();
    }
    const bool want_dh = dhidden_d && rows > 0;
    const int weight_blocks = dweight_d || dbias_d ? (h->vocab + 15) / 16 : 0;
    const int64_t blocks = weight_blocks + (want_dh ? (int64_t)(p.chunks + 3) / 4 * h->texts : 0);
    if (blocks == 0) return GS_OK;
#define GSV_ES(NC)                                                                                                            \
    hipLaunchKernelGGL((k_entry_sums<HT, NC>), dim3((unsigned)blocks), dim3(256), 0, s, hs, ws, grad_d, weights_d, tokens_d,    \
                       p.entries, p.first, h->texts, h->vocab, p.chunk, p.chunks, p.part, p.dimp, (T *)dhidden_d, (T *)dweight_d, \
                       dbias_d, h->bias_type, weight_blocks)
    GSV_BY_CHUNKS(h->dim, GSV_ES)
#undef GSV_ES
    GS_CHECK_LAUNCH();
    if (want_dh) {
        hipLaunchKernelGGL((k_entries_join<HT>), dim3(gs_blocks(rows, 4, 8192)), dim3(256), 0, s, p.first, rows, h->length, h->dim,
                           p.chunk, p.chunks, p.part, p.dimp, (T *)dhidden_d);
        GS_CHECK_LAUNCH();
    }
    return GS_OK;
}

}  // namespace gsv

extern "C" int gs_term_weights_workspace(const gs_vocab_head *h, int32_t tokens, size_t *bytes, size_t *grad_bytes) {
    if (int rc = check_texts(h)) return rc;
    GS_REQUIRE(bytes && grad_bytes, "NULL size pointer");
    const Layout l = layout_of(h);
    gs_arena a{nullptr, 0, 0}, b{nullptr, 0, 0};
    Common c;
    take_common(a, l, h, true, &c);
    const size_t slots = text_slots(h, l);
    a.take<float>(slots * h->vocab);
    if (tokens) a.take<int>(slots * h->vocab);
    take_weight(a, l, h, &c);
    EntryPlan p;
    take_entries(b, h, &p);
    *bytes = a.used, *grad_bytes = b.used;
    return GS_OK;
}

extern "C" int gs_term_weights(const gs_vocab_head *h, const uint8_t *mask_d, float *weights_d, int32_t *tokens_d,
                               void *workspace_d, size_t workspace_bytes, void *stream) {
    if (int rc = check_texts(h)) return rc;
    int cus = 0;
    if (int rc = cu_count(&cus)) return rc;
    const Layout l = layout_of(h);
    gs_arena a{(char *)workspace_d, 0, workspace_bytes};
    Common c;
    take_common(a, l, h, true, &c);
    const size_t slots = text_slots(h, l);
    float *best = a.take<float>(slots * h->vocab);
    int *where = tokens_d ? a.take<int>(slots * h->vocab) : nullptr;
    take_weight(a, l, h, &c);
    if (!a.ok()) {
        gs_set_error("term_weights workspace too small: need %zu bytes, got %zu", a.used, workspace_bytes);
        return GS_ENOSPC;
    }
    if (h->texts == 0) return GS_OK;
    if (int rc = check_data(h)) return rc;
    GS_REQUIRE(weights_d && workspace_d, "NULL weights or workspace");
    const hipStream_t s = gs_stream(stream);
    if (l.rows == 0) {  // texts without tokens
        const int64_t n = (int64_t)h->texts * h->vocab;
        hipLaunchKernelGGL(k_no_tokens, dim3(gs_blocks(n, 256, 8192)), dim3(256), 0, s, n, weights_d, tokens_d);
        GS_CHECK_LAUNCH();
        return GS_OK;
    }
    if (l.cls == kSmall && few_rows_ok(h, l)) {
        const Source hs = hidden_source(h);
        const Operand w = weight_operand(l, c, h);
        const dim3 g((h->vocab + 63) / 64);
#define GSV_FEW(T, TOK)                                                                                                    \
    hipLaunchKernelGGL((k_few_rows<T, TOK>), g, dim3(256), 0, s, hs, mask_d, w, h->bias_d, h->bias_type, h->texts, h->length, \
                       h->vocab, weights_d, tokens_d)
        if (h->type == GS_H_F16) {
            if (tokens_d) GSV_FEW(F16, true);
            else GSV_FEW(F16, false);
        } else {
            if (tokens_d) GSV_FEW(Bf16, true);
            else GSV_FEW(Bf16, false);
        }
#undef GSV_FEW
        GS_CHECK_LAUNCH();
        return GS_OK;
    }
    if (int rc = prepare(h, l, Keep{mask_d, nullptr, 0, h->vocab, l.rows}, c, nullptr, 0, TargetRows{}, TeacherRows{}, s)) return rc;
    {
        const Dims d{l.rows, h->vocab, l.dimp, c.n, 1, 0, 0};
        const Operand hid = hidden_operand(l, c), w = weight_operand(l, c, h);
        const EpiTextMax<true> et{c.bias, c.seg, best, where, h->vocab, nullptr, nullptr};
        const EpiTextMax<false> ef{c.bias, c.seg, best, where, h->vocab, nullptr, nullptr};
        int rc = GS_OK;
#define GSV_TILE(TL, T, NP)                                                                  \
    rc = tokens_d ? launch_product<TL<T, NP, false, false>>(hid, w, d, et, cus, s)             \
                  : launch_product<TL<T, NP, false, false>>(hid, w, d, ef, cus, s)
#define GSV_TILES(T, NP)                                 \
    switch (l.cls) {                                     \
        case kSmall: GSV_TILE(Small, T, NP); break;      \
        case kWide: GSV_TILE(Flat, T, NP); break;        \
        default: GSV_TILE(Large, T, NP); break;          \
    }
        GSV_BY_TYPE(h->type, GSV_TILES)
#undef GSV_TILES
#undef GSV_TILE
        if (rc) return rc;
    }
    const dim3 g(gs_blocks(h->vocab, 1024, 1024), h->texts);
    const int block = token_block(l.cls);
    const Source hs = hidden_source(h), ws = weight_source(h);
#define GSV_TW(TOK, HT)                                                                                                        \
    hipLaunchKernelGGL((k_term_weights<TOK, HT>), g, dim3(256), 0, s, best, where, c.text_first, block, h->vocab, c.rows, h->length, \
                       weights_d, tokens_d, hs, ws, c.bias)
    if (!tokens_d) GSV_TW(false, GS_H_F32);
    else if (h->type == GS_H_F32) GSV_TW(true, GS_H_F32);
    else if (h->type == GS_H_F16) GSV_TW(true, GS_H_F16);
    else GSV_TW(true, GS_H_BF16);
#undef GSV_TW
    GS_CHECK_LAUNCH();
    return GS_OK;
}

extern "C" int gs_term_weights_grad(const gs_vocab_head *h, const float *grad_d, const float *weights_d, const int32_t *tokens_d,
                                    void *dhidden_d, void *dweight_d, void *dbias_d, void *workspace_d, size_t workspace_bytes,
                                    void *stream) {
    if (int rc = check_texts(h)) return rc;
    gs_arena a{(char *)workspace_d, 0, workspace_bytes};
    EntryPlan p;
    take_entries(a, h, &p);
    if (!a.ok()) {
        gs_set_error("term_weights_grad workspace too small: need %zu bytes, got %zu", a.used, workspace_bytes);
        return GS_ENOSPC;
    }
    if (int rc = check_data(h)) return rc;
    GS_REQUIRE((grad_d && weights_d && tokens_d) || h->texts == 0, "NULL gradient, weights or tokens");
    GS_REQUIRE(workspace_d || a.used == 0, "NULL workspace");
    const hipStream_t s = gs_stream(stream);
    if (h->type == GS_H_F32) return run_entries<GS_H_F32>(h, grad_d, weights_d, tokens_d, dhidden_d, dweight_d, dbias_d, p, s);
    if (h->type == GS_H_F16) return run_entries<GS_H_F16>(h, grad_d, weights_d, tokens_d, dhidden_d, dweight_d, dbias_d, p, s);
    return run_entries<GS_H_BF16>(h, grad_d, weights_d, tokens_d, dhidden_d, dweight_d, dbias_d, p, s);
}

// ---------------------------------------------------------------- term weights of a vocabulary in 8 bits

namespace gsv {

// As layout_of, whose unit is 16 bits
Layout layout8_of(const gs_vocab_head *h) {
    const int rows = h->texts * h->length;
    return Layout{rows, (int)round_up(h->dim, kPad8) / 2, 1, (int)round_up(h->vocab, kRowPad), true, class_of(rows)};
}

int check_texts8(const gs_vocab_head *h) {
    if (int rc = check_texts(h)) return rc;
    GS_REQUIRE(h->weight_row_stride % kPad8 == 0 && h->weight_row_stride >= round_up(h->dim, kPad8) && h->weight_row_stride < (1 << 20),
               "weight_row_stride=%lld of 8-bit rows: a multiple of %d, at least dim rounded up to one, below 2^20",
               (long long)h->weight_row_stride, kPad8);
    GS_REQUIRE(h->weight_dim_stride == 1, "weight_dim_stride=%lld of 8-bit rows, which lie on end", (long long)h->weight_dim_stride);
    return GS_OK;
}

// The kept hidden states in 8 bits, where they came from, and the bias.
template <int HT, bool UNIT>
int prepare8(const gs_vocab_head *h, const Layout &l, const Source &hs, const uint8_t *mask_d, const Common &c, float *row_scales, hipStream_t s) {
    if (l.rows <= kPackMost) {
        const int row_blocks = (l.rows + kPackRows - 1) / kPackRows;
        hipLaunchKernelGGL((k_setup_pack8<HT, UNIT>), dim3(row_blocks + l.vocabp / 256), dim3(256), 0, s, hs, mask_d, l.rows, h->texts,
                           row_blocks, 2 * l.dimp, (int8_t *)c.hidden, row_scales, c.seg, c.text_first, c.n, h->bias_d, h->bias_type, h->vocab,
                           l.vocabp, c.bias);
        GS_CHECK_LAUNCH();
        return GS_OK;
    }
    hipLaunchKernelGGL(k_setup, dim3(1 + gs_blocks(l.vocabp, 1024, 1024)), dim3(1024), 0, s, Keep{mask_d, nullptr, 0, h->vocab, l.rows},
                       h->length, c.rows, c.inv, c.seg, c.text_first, c.n, h->bias_d, h->bias_type, h->vocab, l.vocabp, c.bias, nullptr,
                       (int64_t)0);
    GS_CHECK_LAUNCH();
    hipLaunchKernelGGL((k_pack8<HT, UNIT>), dim3(gs_blocks(l.rows, 4, 8192)), dim3(256), 0, s, hs, c.rows, c.n, 2 * l.dimp, (int8_t *)c.hidden,
                       row_scales);
    GS_CHECK_LAUNCH();
    return GS_OK;
}

template <int HT>
int run_terms8(const gs_vocab_head *h, const Layout &l, const float *scales_d, const uint8_t *mask_d, float *weights_d, const Common &c,
               float *best, float *row_scales, int cus, hipStream_t s) {
    using T = typename HVal<HT>::t;
    const Source hs = hidden_source(h);
    if (few8_ok<EpiFewTerms>(l.rows, 2 * l.dimp, h->hidden_dim_stride))
        return launch_few8<T>(hs, mask_d, l.rows, Weight8{(const int8_t *)h->weight_d, h->weight_row_stride, scales_d, h->vocab}, 2 * l.dimp,
                              EpiFewTerms{h->bias_d, h->bias_type, h->texts, h->length, weights_d}, cus, s);
    if (int rc = hs.sd == 1 ? prepare8<HT, true>(h, l, hs, mask_d, c, row_scales, s) : prepare8<HT, false>(h, l, hs, mask_d, c, row_scales, s))
        return rc;
    const Dims d{l.rows, h->vocab, l.dimp, c.n, 1, 0, 0};
    const Operand hid{c.hidden, l.dimp, 0, l.dimp}, w{(const uint16_t *)h->weight_d, h->weight_row_stride / 2, 0, l.dimp};
    const EpiTextMax<false, true> epi{c.bias, c.seg, best, nullptr, h->vocab, row_scales, scales_d};
    int rc = GS_OK;
    switch (l.cls) {
        case kSmall: rc = launch_product<Small<I8, 1, false, false>>(hid, w, d, epi, cus, s); break;
        case kWide: rc = launch_product<Flat<I8, 1, false, false>>(hid, w, d, epi, cus, s); break;
        default: rc = launch_product<Large<I8, 1, false, false>>(hid, w, d, epi, cus, s); break;
    }
    if (rc) return rc;
    hipLaunchKernelGGL((k_term_weights<false, GS_H_F32>), dim3(gs_blocks(h->vocab, 1024, 1024), h->texts), dim3(256), 0, s, best, nullptr,
                       c.text_first, token_block(l.cls), h->vocab, c.rows, h->length, weights_d, nullptr, hs, hs, c.bias);
    GS_CHECK_LAUNCH();
    return GS_OK;
}

void take_terms8(gs_arena &a, const Layout &l, const gs_vocab_head *h, Common *c, float **best, float **row_scales) {
    take_common(a, l, h, true, c);
    *row_scales = a.take<float>(l.rows);
    *best = a.take<float>(text_slots(h, l) * h->vocab);
}

}  // namespace gsv

extern "C" int gs_term_weights8_workspace(const gs_vocab_head *h, size_t *bytes) {
    if (int rc = check_texts8(h)) return rc;
    GS_REQUIRE(bytes, "NULL size pointer");
    const Layout l = layout8_of(h);
    gs_arena a{nullptr, 0, 0};
    Common c;
    float *best, *row_scales;
    if (!few8_ok<EpiFewTerms>(l.rows, 2 * l.dimp, h->hidden_dim_stride)) take_terms8(a, l, h, &c, &best, &row_scales);
    *bytes = a.used;
    return GS_OK;
}

extern "C" int gs_term_weights8(const gs_vocab_head *h, const float *scales_d, const uint8_t *mask_d, float *weights_d, void *workspace_d,
                                size_t workspace_bytes, void *stream) {
    if (int rc = check_texts8(h)) return rc;
    const Layout l = layout8_of(h);
    gs_arena a{(char *)workspace_d, 0, workspace_bytes};
    Common c{};
    float *best = nullptr, *row_scales = nullptr;
    if (!few8_ok<EpiFewTerms>(l.rows, 2 * l.dimp, h->hidden_dim_stride)) take_terms8(a, l, h, &c, &best, &row_scales);
    if (!a.ok()) {
        gs_set_error("term_weights8 workspace too small: need %zu bytes, got %zu", a.used, workspace_bytes);
        return GS_ENOSPC;
    }
    if (h->texts == 0) return GS_OK;
    if (int rc = check_data(h)) return rc;
    GS_REQUIRE(scales_d && weights_d && (workspace_d || a.used == 0), "NULL scales, weights or workspace");
    GS_REQUIRE((uintptr_t)h->weight_d % 16 == 0, "8-bit rows that are not 16-byte aligned");
    const hipStream_t s = gs_stream(stream);
    if (l.rows == 0) {
        const int64_t n = (int64_t)h->texts * h->vocab;
        hipLaunchKernelGGL(k_no_tokens, dim3(gs_blocks(n, 256, 8192)), dim3(256), 0, s, n, weights_d, nullptr);
        GS_CHECK_LAUNCH();
        return GS_OK;
    }
    int cus = 0;
    if (int rc = cu_count(&cus)) return rc;
    if (h->type == GS_H_F32) return run_terms8<GS_H_F32>(h, l, scales_d, mask_d, weights_d, c, best, row_scales, cus, s);
    if (h->type == GS_H_F16) return run_terms8<GS_H_F16>(h, l, scales_d, mask_d, weights_d, c, best, row_scales, cus, s);
    return run_terms8<GS_H_BF16>(h, l, scales_d, mask_d, weights_d, c, best, row_scales, cus, s);
}
