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
//   in 8 bits: maxima over text as above; linear layers with columns of the weight as rows, tokens as columns
//
// Either operand may lie k-major: its tiles are then read from LDS with the transposing
// reads (ds_read_b64_tr_b16), so no matrix is ever transposed in memory.
//
// fp32 operands come as three bf16 planes each (x = p0 + p1 + p2, each the bf16 nearest to
// what is left, 2^-27 of x at most lost) and the product runs over the six plane pairs whose
// product is at least 2^-18 of the largest: what is left out is below 2^-25 of |x||y|, less than
// the rounding of an fp32 product.  (Infinities: split3.)
#pragma once

#include <atomic>

#include "gs_values.h"

namespace gsv {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
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

constexpr int kStep = 64;  // k values per stage: two 16x16x32 products deep, and whole 128-byte lines of [x][k] rows

// A 16-bit matrix.  [x][k]: row x starts at p + x * stride; [k][x]: row k does.  Plane i of an
// fp32 matrix starts `plane` values further along each row.
//
// In blocks: 64 x 64 values are 8 KiB on end, 64 rows of them `stride` values from the next 64; planes follow one another
// along these rows of blocks.  A block holds eight rows at a time, of these the first eight values of each row, then the
// second eight, ...  (The logit gradients, [token][term]: the wave that makes them writes whole lines, either product that
// reads them, along terms or along tokens, copies whole blocks to LDS, and a stage lies in a few pages.)
struct Operand {
    const uint16_t *p;
    int64_t stride;
    int64_t plane;
    int64_t width;  // values of a row (of blocks) that may be read (all planes)
};
constexpr int kBlock = 64, kBlockValues = kBlock * kBlock;
// Where in a block value v of row x is
__host__ __device__ __forceinline__ constexpr int in_block(int x, int v) {
    return (x >> 3) * 512 + (v >> 3) * 64 + (x & 7) * 8 + (v & 7);
}

// Sizes of a product.  Those that depend on the number of kept rows are read from n_d.
struct Dims {
    int32_t r, c, k;
    const int32_t *n_d;
    int32_t dev_r, dev_c, dev_k;  // 1: the size is min(*n_d, the one given)
};

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
// [x][k]: a piece is eight rows of 128 bytes, and slot s of row x holds 16-byte chunk s ^ (x & 7), so that the eight rows
// that one read cycle takes lie in different banks.  (Rows of 64 bytes asked the L2 for half lines: 20% slower.)  [k][x]:
// a piece is 1024 / (2 X) rows of X values, chunks moved in pairs by the k row, so that the rows of a transposing read do.
// The waves take pieces in turn, so that a wave's pieces differ by whole rows and share one offset per lane.
// In blocks: a piece is eight rows of a block as they lie, the rows' odd chunks with their halves of four rows swapped, so
// that a transposing read's four rows of two chunks differ in their banks.
template <int X, bool KM, bool BL, int NW>
struct Loader {
    static constexpr int pieces = X / 8 / NW;
    static constexpr int per = KM ? X / 8 : 8;       // 16-byte chunks of a row
    static constexpr int step = 64 / per * NW;       // rows between a wave's pieces
    static_assert(BL || pieces == 1 || step % (KM ? 16 : 8) == 0, "chunks move alike in all of a wave's pieces");
    static_assert(!BL || NW == 8 || X == kBlock, "a wave's pieces are a block apart, or in one block");
    __device__ __forceinline__ static int offset(const Operand &o, int wave, int lane) {
        if (BL) return wave * 1024 + (lane >> 3) * 128 + ((lane & 7) ^ ((lane >> 1) & 4)) * 16;
        const int row = wave * (64 / per) + lane / per, s = lane % per;
        return (int)(row * o.stride * 2) + (s ^ (KM ? turn<X>(row) << 1 : row & 7)) * 16;
    }
    __device__ __forceinline__ static int gap(const Operand &o) {
        if (BL) return NW < 8 ? NW * 1024 : KM ? kBlockValues * 2 : (int)o.stride * 2;
        return step * (int)o.stride * 2;
    }
    // gap: bytes between a wave's pieces
    __device__ __forceinline__ static void issue(__amdgpu_buffer_rsrc_t r, int gap, int off, int soff, lds_t lds, int wave) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass does not know 16-byte pieces and would leave the kernel out
#pragma unroll
        for (int u = 0; u < pieces; u++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)(lds + ((wave + u * NW) << 10)), 16,
                                                     off + u * gap, soff, 0, 0);
#endif
    }
};

// The next stage of an operand's tile: a buffer that ends with the rows that exist, and an offset into its rows.  The
// buffer of a [x][k] tile stays and the offset moves along its rows (never past them, so the rows that exist are those
// whose own offset lies in the buffer); that of a [k][x] tile moves by the stage's rows.
template <int X, bool KM, bool BL>
struct Cursor {
    const char *p;
    int bytes, soff, rows;
    __device__ __forceinline__ void start(const Operand &o, int x0, int nx, int k, int nk, int plane) {
        const int64_t in = plane * o.plane;
        rows = 0;
        if (BL && KM) {
            p = reinterpret_cast<const char *>(o.p + k / kBlock * o.stride + in + (int64_t)x0 * kBlock);
            bytes = (int)(o.width - in - (int64_t)x0 * kBlock) * 2;
            soff = 0;
        } else if (BL) {
            p = reinterpret_cast<const char *>(o.p + x0 / kBlock * o.stride);
            bytes = (int)((min(nx - x0, X) - 1) / kBlock * o.stride + o.width) * 2;
            soff = (int)(in + (int64_t)k * kBlock) * 2;
        } else if (KM) {
            p = reinterpret_cast<const char *>(o.p + k * o.stride + in + x0);
            rows = nk - k;
            bytes = (int)(o.width - in - x0) * 2;
            soff = 0;
        } else {
            p = reinterpret_cast<const char *>(o.p + x0 * o.stride);
            bytes = (int)((min(nx - x0, X) - 1) * o.stride + o.width) * 2;
            soff = (int)(in + k) * 2;
        }
        uniform();
    }
    // one value per wave, which the compiler does not see through the stream's loop
    __device__ __forceinline__ void uniform() {
        p = reinterpret_cast<const char *>(gs_uniform64(reinterpret_cast<int64_t>(p)));
        bytes = gs_uniform(bytes), soff = gs_uniform(soff), rows = gs_uniform(rows);
    }
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const Operand &o) const {
        return gs_rsrc(p, (uint32_t)(KM && !BL ? (min(rows, kStep) - 1) * (int)(o.stride * 2) + bytes : bytes));
    }
    __device__ __forceinline__ void next(const Operand &o) {
        if (BL) {
            if (KM) p += o.stride * 2;
            else soff += kBlockValues * 2;
        } else if (KM) {
            p += o.stride * (2 * kStep);
            rows -= kStep;
        } else {
            soff += 2 * kStep;
        }
        uniform();
    }
};

// Fragments of 16 rows (columns) x 32 k values, half h of a stage: lane l holds row l & 15, k = 32 h + 8 (l >> 4) .. + 7.
template <int X, bool KM, bool BL, int M>
struct Frags {
    int at[KM && !BL ? M : 2];
    __device__ __forceinline__ void init(int x0, int lane) {  // x0: the wave's first row in the tile
        const int i = lane & 15, q = lane >> 4;
        if (BL && KM) {
            const int odd = (i >> 1) & 1;
            at[0] = (x0 >> 6) * 8192 + q * 1024 + ((x0 >> 3) & 7) * 128 + odd * 128 + ((i >> 2) ^ (odd << 2)) * 16 + (i & 1) * 8;
            at[1] = at[0] ^ 64;  // four rows on
        } else if (BL) {
            at[0] = ((x0 + i) >> 3) * 1024 + q * 128 + ((i & 7) ^ ((q & 1) << 2)) * 16;
            at[1] = at[0] + 512;
        } else if (KM) {
            const int k = 8 * q + (i >> 2);
            const int g = turn<X>(k);
            const int base = k * (X * 2) + ((i >> 1) & 1) * 16 + (i & 1) * 8;
#pragma unroll
            for (int m = 0; m < M; m++) at[m] = base + (((x0 >> 4) + m) ^ g) * 32;
        } else {
            at[0] = (x0 + i) * 128 + (q ^ (i & 7)) * 16;
            at[1] = at[0] ^ 64;
        }
    }
    __device__ __forceinline__ s16x8 read(lds_t lds, int m, int h) const {
        typedef __attribute__((address_space(3))) s16x4 *lp4;
        typedef __attribute__((address_space(3))) s16x8 *lp8;
        if (KM) {
            const int a_at = BL ? at[0] + (m >> 2) * 8192 + (m & 3) * 256 + h * 4096 : at[BL ? 0 : m] + h * 64 * X;
            const int b_at = BL ? at[1] + (m >> 2) * 8192 + (m & 3) * 256 + h * 4096 : a_at + 8 * X;
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp4)(lds + a_at));
            const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp4)(lds + b_at));
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        return *(lp8)(lds + at[h] + m * 2048);
    }
};

// Waits until at most N of this wave's loads are outstanding.
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void tile_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A workgroup's tile: BR x BC over WR x WC waves, NS stages in LDS, OCC waves per SIMD.  RK, CK: R, C lie k-major; CB: C
// lies in blocks.
template <class T, int NP, int BR_, int BC_, int WR_, int WC_, int NS_, int OCC, bool RK, bool CK, bool CB = false>
struct Tile {
    using type = T;
    static constexpr int BR = BR_, BC = BC_, WR = WR_, WC = WC_, NS = NS_, planes = NP;
    static constexpr int waves = WR * WC, threads = 64 * waves, waves_per_simd = OCC;
    static constexpr int MR = BR / WR / 16, MC = BC / WC / 16;
    static constexpr int stage_bytes = (BR + BC) * kStep * 2;
    static constexpr int edge = BR > BC ? BR : BC;
    static constexpr bool r_kmajor = RK, c_kmajor = CK, c_blocks = CB;
};

// What an epilogue reads per row or column of a tile (a bias, a row's softmax sum) comes to LDS with the tile's first
// stage: arrays of TL::edge 32-bit values.  A tile's epilogue runs when NS more stages have been issued, which belong to
// NS more tiles where each has a single one: NS + 1 sets of arrays.
struct SideArray {
    const void *p;  // of the tile's first row or column
    int count;      // values from there on that exist; the others read 0
};

// Where a wave's 16x16 blocks lie: block (i, j) has rows row0 + 16 i + 4 (lane >> 4) + 0..3 and column
// col0 + 16 j + (lane & 15).
struct Place {
    int row0, col0, lane, split;
    int n_r, n_c;
    int r_in, c_in;  // row0 and col0 within the tile
    lds_t sides;
    int edge;
    // side array a's values at in .. in + 3 (of the tile), or the one at in
    __device__ __forceinline__ f32x4 side4(int a, int in) const {
        return *(__attribute__((address_space(3))) f32x4 *)(sides + (a * edge + in) * 4);
    }
    __device__ __forceinline__ float side(int a, int in) const {
        return *(__attribute__((address_space(3))) float *)(sides + (a * edge + in) * 4);
    }
};

// A product's sizes as the device knows them.
struct Shape {
    int nr, nc, nk, tr, tc, steps;
};
template <class TL>
__device__ __forceinline__ Shape shape_of(const Dims &d, int n_dev) {
    Shape s;
    s.nr = d.dev_r ? min(n_dev, d.r) : d.r;
    s.nc = d.dev_c ? min(n_dev, d.c) : d.c;
    s.nk = d.dev_k ? min(n_dev, d.k) : d.k;
    s.tr = (s.nr + TL::BR - 1) / TL::BR;
    s.tc = (s.nc + TL::BC - 1) / TL::BC;
    s.steps = (s.nk + kStep - 1) / kStep;
    return s;
}

// Whether a tile's sums start with the epilogue's side array 0, one value per row (a bias), instead of 0.  Not with fp32
// operands, whose small products are summed first.
template <class TL, class Epi>
constexpr bool starts_with_rows = std::remove_cv_t<std::remove_reference_t<Epi>>::row_bias && TL::planes == 1;

// One product of a launch: tiles [0, tr * tc * parts) of it, each part a range of k.
template <class TL, class Epi>
struct Side {
    using tile = TL;
    using epilogue = Epi;
    static constexpr int set_bytes = Epi::sides * TL::edge * 4;  // of side arrays
    static constexpr int lds_bytes = TL::NS * TL::stage_bytes + (TL::NS + 1) * set_bytes;
    Operand R, C;
    Dims d;
    Epi epi;
};

struct Work {  // a tile: where it lies, which part of k, its first k step and how many
    int r0, c0, part, k0, per;
};
// Tile t.  Eight tiles of rows go with each tile of columns, so that tiles in a row share operands.
template <class TL>
__device__ __forceinline__ Work work_of(const Shape &s, int parts, int t) {
    const int area = s.tr * s.tc, part = t / area, in = t - part * area;
    const int group = in / (8 * s.tc), left = in - group * 8 * s.tc;
    const int tall = min(8, s.tr - group * 8);
    const int k0 = s.steps * part / parts;  // at most 2^22 steps and 128 parts
    return Work{gs_uniform((group * 8 + left % tall) * TL::BR), gs_uniform((left / tall) * TL::BC), gs_uniform(part), gs_uniform(k0),
                gs_uniform(s.steps * (part + 1) / parts - k0)};
}

// What an XCD (blockIdx mod 8) takes of a launch: a contiguous run of either product's tiles, so that what runs at a time in
// an XCD shares operands in its L2, and as much of the long tiles as of the short ones as every other.
struct Share {
    int a0, na, b0, nb;
    __device__ __forceinline__ Share(int ta, int tb, int xcd, int xcds) {
        a0 = (int)((int64_t)ta * xcd / xcds), na = (int)((int64_t)ta * (xcd + 1) / xcds) - a0;
        b0 = (int)((int64_t)tb * xcd / xcds), nb = (int)((int64_t)tb * (xcd + 1) / xcds) - b0;
    }
};

// The stages of a workgroup's tiles, issued one after the other whatever tile they belong to: while a tile's epilogue
// runs, the next one's first stages are on their way.
template <class SA, class SB>
struct Stream {
    using TA = typename SA::tile;
    using TB = typename SB::tile;
    static constexpr bool pair = !std::is_same_v<SA, SB>;
    static constexpr int loads = Loader<TA::BR, TA::r_kmajor, false, TA::waves>::pieces +
                                 Loader<TA::BC, TA::c_kmajor, TA::c_blocks, TA::waves>::pieces;
    Work w;
    int r_off, c_off;     // the lane's
    Cursor<TA::BR, TA::r_kmajor, false> ra;
    Cursor<TA::BC, TA::c_kmajor, TA::c_blocks> ca;
    Cursor<TB::BR, TB::r_kmajor, false> rb;
    Cursor<TB::BC, TB::c_kmajor, TB::c_blocks> cb;
    Share share;
    int t, by;            // the workgroup's tiles: t, t + by, ... of its XCD's share
    int ik, seg, buf, left;
    bool fresh;           // the next stage is its tile's first
    int set;              // of the tile's side arrays

    __device__ __forceinline__ bool in_a() const { return !pair || t < share.na; }
    template <class S>
    __device__ __forceinline__ void sides(const S &side, const Shape &s, lds_t lds, int wave, int lane) const {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
        for (int a = 0; a < S::epilogue::sides; a++) {
            if (wave != a % TA::waves || lane * 4 >= TA::edge) continue;
            const SideArray x = side.epi.side(a, w.r0, w.c0, s);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                gs_rsrc(x.p, (uint32_t)max(x.count, 0) * 4u),
                (__attribute__((address_space(3))) void *)(lds + TA::NS * TA::stage_bytes + set * S::set_bytes + a * TA::edge * 4), 16,
                lane * 16, 0, 0, 0);
        }
#endif
    }
    template <class S, class CR, class CC>
    __device__ __forceinline__ void seek_in(const S &side, const Shape &s, int parts, int at, CR &r, CC &c, int wave, int lane) {
        using TL = typename S::tile;
        w = work_of<TL>(s, parts, at);
        left = w.per * (TL::planes == 3 ? 6 : 1);
        seg = ik = 0;
        r_off = Loader<TL::BR, TL::r_kmajor, false, TL::waves>::offset(side.R, wave, lane);
        c_off = Loader<TL::BC, TL::c_kmajor, TL::c_blocks, TL::waves>::offset(side.C, wave, lane);
        planes(side, s, r, c);
    }
    // To the first stage of plane pair seg
    template <class S, class CR, class CC>
    __device__ __forceinline__ void planes(const S &side, const Shape &s, CR &r, CC &c) {
        constexpr bool three = S::tile::planes == 3;
        r.start(side.R, w.r0, s.nr, w.k0 * kStep, s.nk, three ? plane_r(seg) : 0);
        c.start(side.C, w.c0, s.nc, w.k0 * kStep, s.nk, three ? plane_c(seg) : 0);
    }
    // Moves to tile t, or the next one with stages
    __device__ __forceinline__ void seek(const SA &A, const SB &B, const Shape &a, const Shape &b, int parts, int wave, int lane) {
        for (; t < share.na + share.nb; t += by) {
            if (in_a()) seek_in(A, a, parts, share.a0 + t, ra, ca, wave, lane);
            else seek_in(B, b, 1, share.b0 + t - share.na, rb, cb, wave, lane);
            if (left == 0) continue;
            fresh = true;
            set = set == TA::NS ? 0 : set + 1;
            return;
        }
    }
    template <class S, class CR, class CC>
    __device__ __forceinline__ void issue_in(const S &side, const Shape &s, CR &r, CC &c, lds_t lds, int wave, int lane) {
        using TL = typename S::tile;
        const lds_t to = lds + buf * TL::stage_bytes;
        if (S::epilogue::sides > 0 && fresh) sides(side, s, lds, wave, lane);
        using LR = Loader<TL::BR, TL::r_kmajor, false, TL::waves>;
        using LC = Loader<TL::BC, TL::c_kmajor, TL::c_blocks, TL::waves>;
        LR::issue(r.buffer(side.R), LR::gap(side.R), r_off, r.soff, to, wave);
        LC::issue(c.buffer(side.C), LC::gap(side.C), c_off, c.soff, to + TL::BR * kStep * 2, wave);
        fresh = false;
        if (TL::planes == 3 && ++ik == w.per) {
            ik = 0;
            seg++;
            if (left > 1) planes(side, s, r, c);
        } else {
            r.next(side.R);
            c.next(side.C);
        }
    }
    __device__ __forceinline__ bool issue(lds_t lds, const SA &A, const SB &B, const Shape &a, const Shape &b, int parts, int wave,
                                          int lane) {
        if (t >= share.na + share.nb) return false;
        if (in_a()) issue_in(A, a, ra, ca, lds, wave, lane);
        else issue_in(B, b, rb, cb, lds, wave, lane);
        buf = buf == TA::NS - 1 ? 0 : buf + 1;
        left = gs_uniform(left - 1);
        if (left == 0) {
            t = gs_uniform(t + by);
            seek(A, B, a, b, parts, wave, lane);
        }
        return true;
    }
};

// Parts of k for the first of two products that share a launch: as many as make its tiles as long as the second's, or
// fill `slots` workgroups, at most `most`.  Device code: the sizes are known there alone.
__device__ __forceinline__ int parts_of(int steps, int tiles, int other_steps, int other_tiles, int slots, int most) {
    const int even = other_tiles > 0 ? (steps + other_steps / 2) / max(1, other_steps) : 1;
    const int fill = other_tiles >= slots ? 1 : (slots - other_tiles) / max(1, tiles);
    return max(1, min(most, max(even, fill)));
}

struct Pairing {
    int piece;     // most columns of the second product
    int slots;     // workgroups
    int most;      // parts
    int *parts_d;  // receives the parts (unless there are no rows); NULL: one, and there is no second product
};

// One or two products in a launch, persistent over their tiles.
template <class SA, class SB>
__global__ __launch_bounds__(SA::tile::threads, SA::tile::waves_per_simd) void k_product(SA A, SB B, Pairing pair) {
    using TA = typename SA::tile;
    using TB = typename SB::tile;
    static_assert(SA::lds_bytes == SB::lds_bytes && SA::lds_bytes <= 163840 && TA::MR == TB::MR && TA::MC == TB::MC, "one tile shape per launch");
    extern __shared__ __align__(1024) char smem[];
    const lds_t lds = (lds_t)smem;
    const int lane = gs_lane(), wave = gs_uniform((int)threadIdx.x >> 6);
    const int wr = wave / TA::WC, wc = wave % TA::WC;
    const int n = A.d.n_d ? gs_uniform(*A.d.n_d) : 0;
    const Shape a = shape_of<TA>(A.d, n), b = shape_of<TB>(B.d, B.d.n_d ? gs_uniform(*B.d.n_d) : 0);
    int parts = 1, nb = 0;
    if (pair.parts_d) {
        nb = b.tr * b.tc;
        // from a whole piece's size, so that every piece has the same parts
        parts = parts_of((pair.piece + kStep - 1) / kStep, a.tr * a.tc, b.steps, b.tr * ((pair.piece + TB::BC - 1) / TB::BC),
                         pair.slots, pair.most);
        if (blockIdx.x == 0 && threadIdx.x == 0 && n > 0) *pair.parts_d = parts;
    }
    const int xcds = gridDim.x >= 8 ? 8 : 1, xcd = blockIdx.x % xcds;
    const Share share(a.tr * a.tc * parts, nb, xcd, xcds);

    Stream<SA, SB> st{.share = share};
    st.t = blockIdx.x / xcds;
    st.by = (gridDim.x - xcd + xcds - 1) / xcds;
    st.buf = 0;
    st.set = TA::NS;
    const int first = st.t, by = st.by;
    st.seek(A, B, a, b, parts, wave, lane);
    constexpr int loads = Stream<SA, SB>::loads, NS = TA::NS;
    int ahead = 0;  // stages issued and not yet left behind
#pragma unroll
    for (int s = 0; s < NS - 1; s++) ahead += st.issue(lds, A, B, a, b, parts, wave, lane);
    int buf = 0;

    auto landed = [&]() {  // the oldest of the stages ahead is there, for every wave; and every wave is past the one before
        if (NS > 2 && ahead == NS - 1) wait_loads<(NS > 2 ? NS - 2 : 0) * loads>();
        else wait_loads<0>();
        tile_barrier();
    };
    landed();
    ahead += st.issue(lds, A, B, a, b, parts, wave, lane);
    int set = 0;

    // A tile.  The fragments of a half stage are read while the products of the half before run.  Before a stage's second
    // half the next stage has to have landed, and this one, which every wave holds by then, makes room for another.
    auto run = [&](auto &side, const Work &w, const Shape &s) {
        using TL = typename std::remove_reference_t<decltype(side)>::tile;
        Frags<TL::BR, TL::r_kmajor, false, TL::MR> fr;
        Frags<TL::BC, TL::c_kmajor, TL::c_blocks, TL::MC> fc;
        fr.init(wr * TL::MR * 16, lane);
        fc.init(wc * TL::MC * 16, lane);
        const Place at{w.r0 + wr * TL::MR * 16, w.c0 + wc * TL::MC * 16, lane, w.part, s.nr, s.nc, wr * TL::MR * 16,
                       wc * TL::MC * 16, lds + NS * TL::stage_bytes + set * std::remove_reference_t<decltype(side)>::set_bytes, TL::edge};
        f32x4 acc[TL::MR][TL::MC];
#pragma unroll
        for (int i = 0; i < TL::MR; i++) {
            const f32x4 x = starts_with_rows<TL, decltype(side.epi)> ? at.side4(0, at.r_in + 16 * i + 4 * (lane >> 4))
                                                                     : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < TL::MC; j++) acc[i][j] = x;
        }
        s16x8 fa[2][TL::MR], fb[2][TL::MC];
        auto read = [&](int h) {
            const lds_t from = lds + buf * TL::stage_bytes;
#pragma unroll
            for (int j = 0; j < TL::MC; j++) fb[h][j] = fc.read(from + TL::BR * kStep * 2, j, h);
#pragma unroll
            for (int i = 0; i < TL::MR; i++) fa[h][i] = fr.read(from, i, h);
        };
        auto multiply = [&](int h) {
#pragma unroll
            for (int i = 0; i < TL::MR; i++)
#pragma unroll
                for (int j = 0; j < TL::MC; j++) acc[i][j] = TL::type::mfma(fa[h][i], fb[h][j], acc[i][j]);
        };
        const int total = w.per * (TL::planes == 3 ? 6 : 1);
        if (total > 0) read(0);
        auto stage = [&]() {
            read(1);
            multiply(0);
            buf = buf == NS - 1 ? 0 : buf + 1;
            ahead--;
            landed();
            read(0);  // the last one reads the next tile's fragments, or what is there; nothing uses them
            ahead += st.issue(lds, A, B, a, b, parts, wave, lane);
            multiply(1);
        };
        for (int it = 0; it < total - 1; it++) stage();
        const auto held = side.epi.template before<TL>(at);  // on their way during the last stage
        if (total > 0) stage();
        side.epi.template run<TL>(acc, at, held);
        if (total > 0) set = set == NS ? 0 : set + 1;  // as the stream, which knows tiles with stages alone
    };
    for (int t = first; t < share.na + share.nb; t += by) {
        if constexpr (!std::is_same_v<SA, SB>) {
            if (t < share.na) run(A, work_of<TA>(a, parts, share.a0 + t), a);
            else run(B, work_of<TB>(b, 1, share.b0 + t - share.na), b);
        } else {
            run(A, work_of<TA>(a, 1, share.a0 + t), a);
        }
    }
}

template <class TL>
constexpr int slots_per_cu = TL::waves_per_simd * 4 / TL::waves;

template <class SA, class SB>
int launch_products(const SA &A, const SB &B, const Pairing &pair, int64_t grid, hipStream_t s) {
    using TL = typename SA::tile;
    const void *f = reinterpret_cast<const void *>(&k_product<SA, SB>);
    if (SA::lds_bytes > 65536) {  // once per device
        static std::atomic<uint64_t> set{0};
        int dev = 0;
        GS_CHECK_HIP(hipGetDevice(&dev));
        const uint64_t bit = dev < 64 ? 1ull << dev : 0;
        if (!(set.load(std::memory_order_relaxed) & bit)) {
            GS_CHECK_HIP(hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, SA::lds_bytes));
            set.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    hipLaunchKernelGGL((k_product<SA, SB>), dim3((unsigned)grid), dim3(TL::threads), SA::lds_bytes, s, A, B, pair);
    GS_CHECK_LAUNCH();
    return GS_OK;
}

// Launches a product on as many workgroups as run at a time.
template <class TL, class Epi>
int launch_product(const Operand &R, const Operand &C, const Dims &d, const Epi &epi, int cus, hipStream_t s) {
    const int64_t tiles = (int64_t)((d.r + TL::BR - 1) / TL::BR) * ((d.c + TL::BC - 1) / TL::BC);
    const int64_t slots = (int64_t)slots_per_cu<TL> * cus;
    if (tiles <= 0) return GS_OK;
    const Side<TL, Epi> A{R, C, d, epi};
    return launch_products(A, A, Pairing{0, 0, 1, nullptr}, tiles < slots ? tiles : slots, s);
}

// Two: the first in parts of its k, the second of columns that are the first's k, a piece of at most `piece` of them.
template <class TA, class TB, class EA, class EB>
int launch_pair(const Operand &Ra, const Operand &Ca, const Dims &da, const EA &ea, const Operand &Rb, const Operand &Cb,
                const Dims &db, const EB &eb, int piece, int most, int *parts_d, int cus, hipStream_t s) {
    const int slots = slots_per_cu<TA> * cus;
    return launch_products(Side<TA, EA>{Ra, Ca, da, ea}, Side<TB, EB>{Rb, Cb, db, eb}, Pairing{piece, slots, most, parts_d}, slots, s);
}

}  // namespace gsv
