// The matrix product of the vocabulary head, one kernel for all of its uses.
//
// acc[r][c] = sum_k R[r][k] * C[c][k], 16-bit operands, fp32 sums, for a tile of BR x BC;
// what happens to a tile is the epilogue's business and stays in registers.
//
//   use               rows r        columns c      k         R in memory   C in memory
//   softmax sums      terms         tokens         dim       [r][k]        [c][k]
//   logit gradients   terms         tokens         dim       [r][k]        [c][k]
//   maxima over text  tokens        terms          dim       [r][k]        [c][k]
//   dW                dim           terms          tokens    [k][r]        [k][c]
//   dH                dim           tokens         terms     [k][r]        [c][k]
//
// Either operand may lie k-major: its tiles are then read from LDS with the transposing
// reads (ds_read_b64_tr_b16), so no matrix is ever transposed in memory.
//
// fp32 operands come as three bf16 planes each (x = p0 + p1 + p2, each the bf16 nearest to
// what is left, 2^-27 of x at most lost) and the product runs over the six plane pairs whose
// product is at least 2^-18 of the largest: what is left out is below 2^-25 of |x||y|, less than
// the rounding of an fp32 product.
#pragma once

#include "gs_common.h"

namespace gsv {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char *lds_t;

struct Bf16 {
    using store_t = __bf16;
    __device__ __forceinline__ static f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                       c, 0, 0, 0);
    }
};
struct F16 {
    using store_t = _Float16;
    __device__ __forceinline__ static f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c,
                                                      0, 0, 0);
    }
};

constexpr int kStep = 32;  // k values per stage: one 16x16x32 product deep

// A 16-bit matrix.  [x][k]: row x starts at p + x * stride; [k][x]: row k does.  Plane i of an
// fp32 matrix starts `plane` values further along each row.
struct Operand {
    const uint16_t *p;
    int64_t stride;
    int64_t plane;
    int64_t width;  // values of a row that may be read (all planes)
};

// Sizes of a product.  Those that depend on the number of kept rows are read from n_d.
struct Dims {
    int32_t r, c, k;
    const int32_t *n_d;
    int32_t dev_r, dev_c, dev_k;  // 1: the size is min(*n_d, the one given)
    int32_t split;                // parts of k, each a tile of its own; 0: as many as fill `slots` workgroups,
    int32_t slots, most;          //   at most `most` (parts_of)
};

// Parts of k for a product of tr x ceil(c / bc) tiles.  Device code: c is known there alone.
__device__ __forceinline__ int parts_of(int c, int tr, int bc, int slots, int most) {
    return max(1, min(most, slots / max(1, tr * ((c + bc - 1) / bc))));
}

// The plane pairs, smallest products first, so that they are summed before the sum is large: (2,0) (0,2) (1,1) (1,0)
// (0,1) (0,0).
__device__ __forceinline__ int plane_r(int s) { return (0x001102 >> (4 * s)) & 15; }
__device__ __forceinline__ int plane_c(int s) { return (0x010120 >> (4 * s)) & 15; }

// By what a k row's 16-value blocks are moved (XOR) in a [k][x] tile of X values a row: rows 0..3 and 8..11 of a
// transposing read differ (of 64 values, rows 0..3).
template <int X>
__device__ __forceinline__ int turn(int k) {
    return X >= 128 ? (k & 3) | ((k >> 1) & 4) : k & 3;
}

// Issues one stage's 1 KiB pieces of an operand that belong to this wave, straight to LDS.
// [x][k]: a piece is 16 rows of 64 bytes, and slot s of row x holds 16-byte chunk s ^ (x >> 1 & 3), so that the
// eight rows that one read cycle takes lie in different banks.  [k][x]: a piece is 1024 / (2 X) rows of X values,
// chunks moved in pairs by the k row, so that the four k rows of a transposing read do.
template <int X, bool KM, int NW>
struct Loader {
    static constexpr int pieces = X / 16 / NW;
    int off[pieces];
    __device__ __forceinline__ void init(const Operand &o, int wave, int lane) {
#pragma unroll
        for (int u = 0; u < pieces; u++) {
            const int at = ((wave * pieces + u) << 6) + lane;  // 16-byte slot of the tile
            if (KM) {
                constexpr int per = X / 8;
                const int k = at / per, s = at % per;
                off[u] = (int)(k * o.stride * 2) + (s ^ (turn<X>(k) << 1)) * 16;
            } else {
                const int x = at >> 2, s = at & 3;
                off[u] = (int)(x * o.stride * 2) + (s ^ ((x >> 1) & 3)) * 16;
            }
        }
    }
    __device__ __forceinline__ void issue(__amdgpu_buffer_rsrc_t r, lds_t lds, int soff, int wave) const {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass does not know 16-byte pieces and would leave the kernel out
#pragma unroll
        for (int u = 0; u < pieces; u++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)(lds + ((wave * pieces + u) << 10)),
                                                     16, off[u], soff, 0, 0);
#endif
    }
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc64(const uint16_t *p, int64_t values) {
    const int64_t b = values <= 0 ? 0 : values * 2;
    return gs_rsrc(p, (uint32_t)(b > 0x7FFFFFF0ll ? 0x7FFFFFF0ll : b));
}

// The buffer of one stage: [x][k] tiles keep one for all k (the offset moves), [k][x] tiles move it.
template <bool KM>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t stage_rsrc(const Operand &o, int64_t x0, int64_t nx, int64_t k,
                                                             int64_t nk, int plane) {
    if (KM) return rsrc64(o.p + k * o.stride + plane * o.plane + x0, (nk - k - 1) * o.stride + o.width - plane * o.plane - x0);
    return rsrc64(o.p + x0 * o.stride, (nx - x0 - 1) * o.stride + o.width);
}

// Fragments of 16 rows (columns) x 32 k values: lane l holds row l & 15, k = 8 (l >> 4) .. + 7.
template <int X, bool KM, int M>
struct Frags {
    int at[KM ? M : 1];
    __device__ __forceinline__ void init(int x0, int lane) {  // x0: the wave's first row in the tile
        if (KM) {
            const int i = lane & 15, q = lane >> 4;
            const int k = 8 * q + (i >> 2);
            const int g = turn<X>(k);
            const int base = k * (X * 2) + ((i >> 1) & 1) * 16 + (i & 1) * 8;
#pragma unroll
            for (int m = 0; m < M; m++) at[m] = base + (((x0 >> 4) + m) ^ g) * 32;
        } else {
            const int i = lane & 15, q = lane >> 4;
            at[0] = (x0 + i) * 64 + (q ^ ((i >> 1) & 3)) * 16;
        }
    }
    __device__ __forceinline__ s16x8 read(lds_t lds, int m) const {
        typedef __attribute__((address_space(3))) s16x4 *lp4;
        typedef __attribute__((address_space(3))) s16x8 *lp8;
        if (KM) {
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp4)(lds + at[m]));
            const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp4)(lds + at[m] + 4 * X * 2));
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        return *(lp8)(lds + at[0] + m * 1024);
    }
};

// Waits until at most N of this wave's loads are outstanding.
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void tile_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

template <class T, int NP, int BR_, int BC_, int WR_, int WC_, int NS_, bool RK, bool CK>
struct Tile {
    using type = T;
    static constexpr int BR = BR_, BC = BC_, WR = WR_, WC = WC_, NS = NS_, planes = NP;
    static constexpr int waves = WR * WC, threads = 64 * waves;
    static constexpr int MR = BR / WR / 16, MC = BC / WC / 16;
    static constexpr int stage_bytes = (BR + BC) * 64;
    static constexpr int lds_bytes = NS * stage_bytes;
    static constexpr bool r_kmajor = RK, c_kmajor = CK;
};

// Where a wave's 16x16 blocks lie: block (i, j) has rows row0 + 16 i + 4 (lane >> 4) + 0..3 and column
// col0 + 16 j + (lane & 15).
struct Place {
    int row0, col0, lane, split;
    int n_r, n_c;
};

// Persistent over tiles.  Workgroups of one XCD (blockIdx mod 8) take a contiguous run of tiles, eight tiles of
// rows to each tile of columns, so that what runs at a time in an XCD shares operands in its L2.
template <class TL, class Epi>
__global__ __launch_bounds__(TL::threads, 2) void k_product(Operand R, Operand C, Dims d, Epi epi) {
    extern __shared__ __align__(1024) char smem[];
    const lds_t lds = (lds_t)smem;
    const int lane = gs_lane(), wave = gs_uniform((int)threadIdx.x >> 6);
    const int wr = wave / TL::WC, wc = wave % TL::WC;
    const int n_dev = d.n_d ? gs_uniform(*d.n_d) : 0;
    const int nr = d.dev_r ? min(n_dev, d.r) : d.r, nc = d.dev_c ? min(n_dev, d.c) : d.c;
    const int nk = d.dev_k ? min(n_dev, d.k) : d.k;
    const int tr = (nr + TL::BR - 1) / TL::BR, tc = (nc + TL::BC - 1) / TL::BC;
    const int steps = (nk + kStep - 1) / kStep;
    const int split = d.split ? d.split : parts_of(nc, tr, TL::BC, d.slots, d.most);
    const int64_t tiles = (int64_t)tr * tc * split;

    Loader<TL::BR, TL::r_kmajor, TL::waves> lr;
    Loader<TL::BC, TL::c_kmajor, TL::waves> lc;
    lr.init(R, wave, lane);
    lc.init(C, wave, lane);
    Frags<TL::BR, TL::r_kmajor, TL::MR> fr;
    Frags<TL::BC, TL::c_kmajor, TL::MC> fc;
    fr.init(wr * TL::MR * 16, lane);
    fc.init(wc * TL::MC * 16, lane);
    constexpr int loads = decltype(lr)::pieces + decltype(lc)::pieces;

    const int xcds = gridDim.x >= 8 ? 8 : 1;
    const int xcd = blockIdx.x % xcds, slot = blockIdx.x / xcds;
    const int slots = (gridDim.x - xcd + xcds - 1) / xcds;
    const int64_t first = tiles * xcd / xcds, last = tiles * (xcd + 1) / xcds;
    for (int64_t t = first + slot; t < last; t += slots) {
        const int sp = (int)(t / ((int64_t)tr * tc));
        const int in = (int)(t - (int64_t)sp * tr * tc);
        const int group = in / (8 * tc), left = in - group * 8 * tc;
        const int tall = min(8, tr - group * 8);
        const int r0 = (group * 8 + left % tall) * TL::BR, c0 = (left / tall) * TL::BC;
        const int k_lo = (int)((int64_t)steps * sp / split), k_hi = (int)((int64_t)steps * (sp + 1) / split);
        const int per = k_hi - k_lo;
        const int total = per * (TL::planes == 3 ? 6 : 1);

        f32x4 acc[TL::MR][TL::MC];
#pragma unroll
        for (int i = 0; i < TL::MR; i++)
#pragma unroll
            for (int j = 0; j < TL::MC; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

        const auto r_all = stage_rsrc<false>(R, r0, nr, 0, 0, 0);
        const auto c_all = stage_rsrc<false>(C, c0, nc, 0, 0, 0);
        int ik = 0, iseg = 0, ibuf = 0;  // the next stage to issue
        auto issue = [&]() {
            const int pr = TL::planes == 3 ? plane_r(iseg) : 0, pc = TL::planes == 3 ? plane_c(iseg) : 0;
            const int k = (k_lo + ik) * kStep;
            const lds_t to = lds + ibuf * TL::stage_bytes;
            if (TL::r_kmajor) lr.issue(stage_rsrc<true>(R, r0, 0, k, nk, pr), to, 0, wave);
            else lr.issue(r_all, to, (int)(pr * R.plane + k) * 2, wave);
            if (TL::c_kmajor) lc.issue(stage_rsrc<true>(C, c0, 0, k, nk, pc), to + TL::BR * 64, 0, wave);
            else lc.issue(c_all, to + TL::BR * 64, (int)(pc * C.plane + k) * 2, wave);
            if (++ik == per) {
                ik = 0;
                iseg++;
            }
            ibuf = ibuf == TL::NS - 1 ? 0 : ibuf + 1;
        };
        tile_barrier();  // the last tile's reads are done
        const int ahead = min(TL::NS - 1, total);
        for (int s = 0; s < ahead; s++) issue();
        int buf = 0;
        for (int it = 0; it < total; it++) {
            // stage `it` has landed once only the later ones issued so far are outstanding
            if (it + TL::NS - 1 <= total) wait_loads<(TL::NS - 2) * loads>();
            else wait_loads<0>();
            tile_barrier();
            if (it + TL::NS - 1 < total) issue();
            const lds_t at = lds + buf * TL::stage_bytes;
            s16x8 a[TL::MR], b[TL::MC];
#pragma unroll
            for (int j = 0; j < TL::MC; j++) b[j] = fc.read(at + TL::BR * 64, j);
#pragma unroll
            for (int i = 0; i < TL::MR; i++) a[i] = fr.read(at, i);
#pragma unroll
            for (int i = 0; i < TL::MR; i++)
#pragma unroll
                for (int j = 0; j < TL::MC; j++) acc[i][j] = TL::type::mfma(a[i], b[j], acc[i][j]);
            buf = buf == TL::NS - 1 ? 0 : buf + 1;
        }
        const Place at{r0 + wr * TL::MR * 16, c0 + wc * TL::MC * 16, lane, sp, nr, nc};
        epi.template run<TL>(acc, at);
    }
}

// Launches a product on at most two workgroups per CU.
template <class TL, class Epi>
int launch_product(const Operand &R, const Operand &C, const Dims &d, const Epi &epi, int cus, hipStream_t s) {
    const int64_t tiles = (int64_t)((d.r + TL::BR - 1) / TL::BR) * ((d.c + TL::BC - 1) / TL::BC) *
                          (d.split ? d.split : d.most);
    if (tiles <= 0) return GS_OK;
    if (TL::lds_bytes > 65536)
        GS_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(&k_product<TL, Epi>),
                                         hipFuncAttributeMaxDynamicSharedMemorySize, TL::lds_bytes));
    const int per_cu = TL::lds_bytes > 81920 ? 1 : 2;
    const int64_t grid = tiles < (int64_t)per_cu * cus ? tiles : (int64_t)per_cu * cus;
    hipLaunchKernelGGL((k_product<TL, Epi>), dim3((unsigned)grid), dim3(TL::threads), TL::lds_bytes, s, R, C, d, epi);
    GS_CHECK_LAUNCH();
    return GS_OK;
}

}  // namespace gsv
