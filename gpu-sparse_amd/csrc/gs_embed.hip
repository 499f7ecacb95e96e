// Token lookup, the encoder's first layer, and its gradient:
//   gs_embed_tokens        out[n] = scale * W[id of n]
//   gs_embed_tokens_grad   dW[v] = scale * sum of g[n] over the n whose id is v
// The gradient sorts the tokens by id, stably and without an atomic that decides an order, and sums runs of equal ids: every
// sum has one order, and each row of dW is written once, zeros included.
#include "gs_int8.h"

namespace gsv {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// N values on end of a table's or a gradient's row, aligned as single values are
template <class T, int N>
struct Piece {
    typedef T vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    vec v;
};

struct Ids {
    const void *p;
    int bytes;
    __device__ __forceinline__ int64_t at(int64_t n) const { return bytes == 8 ? ((const int64_t *)p)[n] : ((const int32_t *)p)[n]; }
};

// ---------------------------------------------------------------- lookup

// A thread takes U pieces of N values, 256 apart: all ids first, then all rows, so that their loads are on their way together.
// TAIL: a row's last piece is not whole.  Bytes bound it: 16384 rows of 768 16-bit values 8.5 us, from 8 bits 9.0; 262144 rows of 1024,
// 128003 ids, 170 (537 MB written; of 537 read, 108 of different rows, 329 come from beyond the L2 caches), or 154 where the kernel before
// it leaves the caches alone.
template <class T, class O, int N, int U, bool TAIL>
__global__ __launch_bounds__(256) void k_embed(Ids ids, const T *table, int64_t stride, const float *scales, int vocab, int dim, uint32_t pieces,
                                               int64_t total, float scale, O *out) {
    const int64_t base = (int64_t)blockIdx.x * (256 * U), n0 = base / pieces;
    const uint32_t p0 = (uint32_t)(base - n0 * pieces), most = (uint32_t)min((int64_t)(256 * U), total - base) - 1;
    typename Piece<T, N>::vec x[U];
    float by[U];
    uint32_t row[U], d[U];
    int64_t id[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t at = p0 + min(u * 256 + threadIdx.x, most);  // those past the last one take it again, and write nothing
        row[u] = at / pieces;
        d[u] = (at - row[u] * pieces) * N;
        id[u] = ids.at(n0 + row[u]);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const bool in = id[u] >= 0 && id[u] < vocab;
        const int64_t v = in ? id[u] : 0;
        const T *from = table + v * stride + d[u];
        if (!TAIL || d[u] + N <= dim) {
            x[u] = reinterpret_cast<const Piece<T, N> *>(from)->v;
        } else {
#pragma unroll
            for (int e = 0; e < N; e++) x[u][e] = d[u] + e < dim ? from[e] : (T)0;
        }
        by[u] = scales ? scales[v] : scale;
        row[u] = in ? row[u] : ~row[u];
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (u * 256 + threadIdx.x > most) break;
        const bool in = (int32_t)row[u] >= 0;
        Piece<O, N> y;
#pragma unroll
        for (int e = 0; e < N; e++) y.v[e] = in ? (O)(scales ? (float)x[u][e] * by[u] * scale : (float)x[u][e] * by[u]) : (O)0.f;
        O *to = out + (n0 + (in ? row[u] : ~row[u])) * dim + d[u];
        if (!TAIL || d[u] + N <= dim) {
            *reinterpret_cast<Piece<O, N> *>(to) = y;
        } else {
#pragma unroll
            for (int e = 0; e < N; e++)
                if (d[u] + e < dim) to[e] = y.v[e];
        }
    }
}

// Tables whose rows are not on end: a value at a time
template <class T>
__global__ __launch_bounds__(256) void k_embed_strided(Ids ids, const T *table, int64_t stride, int64_t dim_stride, int vocab, int dim,
                                                       int64_t total, float scale, T *out) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t n = i / dim, id = ids.at(n);
        out[i] = id < 0 || id >= vocab ? (T)0.f : (T)((float)table[id * stride + (i - n * dim) * dim_stride] * scale);
    }
}

// ---------------------------------------------------------------- order

// Tokens sorted by id: order[e], the token of entry e, ascending within an id, and start[v], the first entry of id v (start[vocab]:
// how many there are).  The ids are split into kRanges ranges of 2^shift ids.  One workgroup orders a range; it finds its tokens
// among all ids itself (16384 tokens: 14 us, a launch), or, of more, in segments that k_split has sorted by range (17, two; 262144
// tokens 31, and 270 where all hold one id: a range is one workgroup's, at 1 ns a token).
constexpr int kRanges = 256, kSegs = 1024;
constexpr int kSplitThreads = 512, kSplitWaves = kSplitThreads / 64, kSegTokens = 1024;  // of a segment, at least
// A wave of k_order counts ids on its own, in at most so many bytes of LDS for all waves: fewer waves where ranges are wide.  Beside
// the counts lie the tokens that a wave has found itself, of 1024 that it looks through.
constexpr int kOrderLds = 128 * 1024, kDirectLds = 64 * 1024, kOrderMost = 148 * 1024, kDirectWave = 1024;
__host__ __device__ inline int order_waves(int lds, int shift) {
    const int room = lds / 4 >> shift;
    return room < 16 ? room : 16;
}

struct Tokens {
    Ids ids;
    int64_t n, padding;
    int vocab, shift, ranges;
    // token n's id, -1 where it is not kept
    __device__ __forceinline__ int id(int64_t n) const {
        uint32_t v;
        bool far = false;
        if (ids.bytes == 8) {
            const uint2 x = ((const uint2 *)ids.p)[n];
            v = x.x, far = x.y != 0;
        } else {
            v = ((const uint32_t *)ids.p)[n];
        }
        return far || v >= (uint32_t)vocab || v == (uint32_t)padding ? -1 : (int)v;
    }
};

// Of the lanes that are on: how many before this one hold the same key of `bits` bits, and how many do in all.
__device__ __forceinline__ void same_key(uint32_t key, bool on, int bits, int &rank, int &all) {
    const uint64_t of = __ballot(on);
    uint32_t lo = (uint32_t)of, hi = (uint32_t)(of >> 32);
#pragma unroll
    for (int b = 0; b < 12; b++) {
        if (b >= bits) break;
        const uint32_t mine = 0u - ((key >> b) & 1);
        const uint64_t m = __ballot(mine != 0);
        lo &= ~(mine ^ (uint32_t)m), hi &= ~(mine ^ (uint32_t)(m >> 32));
    }
    const uint64_t same = (uint64_t)hi << 32 | lo;
    rank = __popcll(same & gs_lanemask_lt());
    all = __popcll(same);
}
// Adds the lanes that are on to their keys' counts.  A few keys are counted together first, since adds to one place wait for each
// other.
__device__ __forceinline__ void add_keys(int *count, int key, bool on) {
    uint64_t left = __ballot(on);
#pragma unroll
    for (int k = 0; k < 3; k++) {
        if (!left) return;
        const int first = __builtin_ctzll(left), its = __builtin_amdgcn_readlane(key, first);
        const uint64_t same = __ballot(key == its) & left;
        if (gs_lane() == first) atomicAdd(count + its, __popcll(same));
        left &= ~same;
    }
    if (left >> gs_lane() & 1) atomicAdd(count + key, 1);
}

// Exclusive prefix sums over `n` ints in LDS by a workgroup of W waves, n at most 64 W * 4; returns their total.
template <int W>
__device__ __forceinline__ int block_prefix(int *x, int n, int *wave_sums) {
    const int tid = threadIdx.x, lane = gs_lane(), wave = tid >> 6, per = (n + 64 * W - 1) / (64 * W);
    int v[4], sum = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const int i = tid * per + e;
        v[e] = e < per && i < n ? x[i] : 0;
        sum += v[e];
    }
    const int inc = (int)gs_wave_incl_scan((uint32_t)sum);
    if (lane == 63) wave_sums[wave] = inc;
    __syncthreads();
    int at = inc - sum, total = 0;
    for (int w = 0; w < W; w++) {
        if (w < wave) at += wave_sums[w];
        total += wave_sums[w];
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const int i = tid * per + e;
        if (e < per && i < n) x[i] = at;
        at += v[e];
    }
    __syncthreads();
    return total;
}

// A segment's tokens sorted by range, in order within a range.  pos[segment]: token; low[segment]: the id's bits within its range;
// counts[range][segment], begin[range][segment].
__global__ __launch_bounds__(kSplitThreads) void k_split(Tokens t, int64_t seg_size, int segs, uint32_t *pos, uint16_t *low, int *counts,
                                                         int *begin) {
    __shared__ int count[kSplitWaves][kRanges], first[kRanges], wave_sums[kSplitWaves];
    const int tid = threadIdx.x, lane = gs_lane(), wave = tid >> 6;
    const int64_t s0 = blockIdx.x * seg_size, s1 = min(t.n, s0 + seg_size);
    const int64_t per = (seg_size + kSplitWaves - 1) / kSplitWaves, a = min(s1, s0 + wave * per), b = min(s1, a + per);
    for (int r = lane; r < kRanges; r += 64) count[wave][r] = 0;
    gs_wave_sync();
    for (int64_t n = a + lane; n < b; n += 64) {
        const int id = t.id(n);
        add_keys(count[wave], id >> t.shift, id >= 0);
    }
    __syncthreads();
    if (tid < kRanges) {
        int sum = 0;
        for (int w = 0; w < kSplitWaves; w++) sum += count[w][tid];
        first[tid] = sum;
        counts[(int64_t)tid * segs + blockIdx.x] = sum;
    }
    __syncthreads();
    block_prefix<kSplitWaves>(first, kRanges, wave_sums);
    if (tid < kRanges) {
        int at = first[tid];
        begin[(int64_t)tid * segs + blockIdx.x] = at;
        for (int w = 0; w < kSplitWaves; w++) {
            const int c = count[w][tid];
            count[w][tid] = at;
            at += c;
        }
    }
    __syncthreads();
    for (int64_t n0 = a; n0 < b; n0 += 64) {
        const int64_t n = n0 + lane;
        const int id = n < b ? t.id(n) : -1;
        const bool on = id >= 0;
        const int r = on ? id >> t.shift : 0;
        int rank, all;
        same_key(r, on, 8, rank, all);
        const int at = count[wave][r];
        gs_wave_sync();
        if (on) {
            pos[s0 + at + rank] = (uint32_t)n;
            low[s0 + at + rank] = (uint16_t)(id & ((1 << t.shift) - 1));
            if (rank == 0) count[wave][r] = at + all;
        }
        gs_wave_sync();
    }
}

struct Sorted {
    uint32_t *order;  // [entry]: token
    int *id;          // [entry]
    int *start;       // [vocab + 1]
};

// SPLIT: from k_split's segments.
template <bool SPLIT>
__global__ __launch_bounds__(1024) void k_order(Tokens t, int64_t seg_size, int segs, const uint32_t *pos, const uint16_t *low, const int *counts,
                                                const int *begin, Sorted o) {
    extern __shared__ __align__(16) char smem[];
    __shared__ int wave_sums[16], seg_at[SPLIT ? kSegs + 1 : 1], seg_from[SPLIT ? kSegs : 1], before_s;
    int *count = reinterpret_cast<int *>(smem);  // [waves][width]
    const int tid = threadIdx.x, lane = gs_lane(), wave = tid >> 6;
    const int g = blockIdx.x, width = 1 << t.shift, id0 = g << t.shift;
    const int waves = order_waves(SPLIT ? kOrderLds : kDirectLds, t.shift);
    for (int i = tid; i < waves * width; i += 1024) count[i] = 0;
    if (tid == 0) before_s = 0;
    __syncthreads();
    int64_t n = t.n;
    if (SPLIT) {
        if (tid < segs) seg_at[tid] = counts[(int64_t)g * segs + tid], seg_from[tid] = begin[(int64_t)g * segs + tid];
        int before = 0;
        const int cells = g * segs;  // a whole number of fours where that matters
#pragma unroll 8
        for (int i = tid * 4; i + 3 < cells; i += 4096) {
            const i32x4 c = *reinterpret_cast<const i32x4 *>(counts + i);
            before += c[0] + c[1] + c[2] + c[3];
        }
        if (tid < (cells & 3)) before += counts[(cells & ~3) + tid];
        before = (int)gs_wave_sum((uint32_t)before);
        if (lane == 0) atomicAdd(&before_s, before);
        __syncthreads();
        n = block_prefix<16>(seg_at, segs, wave_sums);
        if (tid == 0) seg_at[segs] = (int)n;
        __syncthreads();
    }
    // A wave takes entries a to b of the range (SPLIT), or lists those of its tokens that are of the range: id within the range and
    // token, in order.
    const int64_t per = (n + waves - 1) / waves, a = wave < waves ? min(n, wave * per) : n, b = min(n, a + per);
    uint32_t *mine = reinterpret_cast<uint32_t *>(count + (waves + 1) * width) + wave * kDirectWave;
    int m = 0;
    if (SPLIT) {
        m = (int)(b - a);
    } else if (a < b) {
        constexpr int kRounds = kDirectWave / 64;
        int id[kRounds], below = 0;
#pragma unroll
        for (int k = 0; k < kRounds; k++) id[k] = t.id(min(a + k * 64 + lane, b - 1));
#pragma unroll
        for (int k = 0; k < kRounds; k++) {
            const int in = k * 64 + lane;
            if (in >= b - a) id[k] = -1;
            below += id[k] >= 0 && id[k] < id0;
            const bool on = id[k] >= 0 && id[k] >> t.shift == g;
            const uint64_t some = __ballot(on);
            if (!some) continue;
            if (on) {
                const int key = id[k] - id0;
                mine[m + __popcll(some & gs_lanemask_lt())] = (uint32_t)key << 10 | in;
            }
            m += __popcll(some);
        }
        below = (int)gs_wave_sum((uint32_t)below);
        if (lane == 0) atomicAdd(&before_s, below);
    }
    gs_wave_sync();
    // f(key, token, on) for the wave's entries, 64 at a time, kAhead rounds' loads on their way together.  An entry's
    // segment is the last that starts at or before it, searched for where ranges hold few entries a segment, else walked to.
    constexpr int kAhead = SPLIT ? 8 : 1;
    const bool walk = SPLIT && n >= segs * 32;
    int key[kAhead], seg;
    uint32_t token[kAhead];
    const auto search = [&](int64_t e) {
        int lo = 0, hi = segs;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (seg_at[mid] <= e) lo = mid;
            else hi = mid;
        }
        return lo;
    };
    const auto fetch = [&](int e0) {
        if constexpr (SPLIT) {
            int64_t at[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                const int64_t e = a + min(e0 + k * 64 + lane, m - 1);
                if (walk) {
                    while (seg_at[seg + 1] <= e) seg++;
                } else {
                    seg = search(e);
                }
                at[k] = seg * seg_size + seg_from[seg] + (e - seg_at[seg]);
            }
#pragma unroll
            for (int k = 0; k < kAhead; k++) key[k] = low[at[k]], token[k] = pos[at[k]];
        } else {
            const uint32_t x = mine[min(e0 + lane, m - 1)];
            key[0] = x >> 10, token[0] = (uint32_t)a + (x & 1023);
        }
    };
    const auto each = [&](bool again, auto &&f) {
        if (SPLIT && walk && m > 0) seg = search(a + min(lane, m - 1));
        for (int e0 = 0; e0 < m; e0 += kAhead * 64) {
            if (!again || m > kAhead * 64) fetch(e0);
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                if (e0 + k * 64 >= m) break;
                f(key[k], token[k], e0 + k * 64 + lane < m);
                gs_wave_sync();
            }
        }
    };
    each(false, [&](int key, uint32_t, bool on) { add_keys(count + wave * width, key, on); });
    __syncthreads();
    // over the waves, then over the ids
    int *first = count + waves * width;
    for (int v = tid; v < width; v += 1024) {
        int sum = 0;
        for (int w = 0; w < waves; w++) {
            const int c = count[w * width + v];
            count[w * width + v] = sum;
            sum += c;
        }
        first[v] = sum;
    }
    __syncthreads();
    const int total = block_prefix<16>(first, width, wave_sums), base = before_s;
    for (int v = tid; v < width && id0 + v < t.vocab; v += 1024) o.start[id0 + v] = base + first[v];
    if (tid == 0 && g == t.ranges - 1) o.start[t.vocab] = base + total;
    for (int i = tid; i < waves * width; i += 1024) count[i] += base + first[i & (width - 1)];
    __syncthreads();
    each(true, [&](int key, uint32_t token, bool on) {
        int rank, all;
        same_key(key, on, t.shift, rank, all);
        int *next = &count[wave * width + key];
        const int at = *next;
        gs_wave_sync();
        if (on) {
            o.order[at + rank] = token;
            o.id[at + rank] = id0 + key;
            if (rank == 0) *next = at + all;
        }
    });
}

// ---------------------------------------------------------------- sums

// A chunk of entries and a slice of 64 N columns are a wave's: it adds the rows of one id after the other in fp32.  A sum whose
// id has all its entries in the chunk is a row of dW; the others are parts: part[chunk][0] of the id that came from before,
// part[chunk][1] of the one that started here.  More waves write the zeros of ids without an entry.
//
// STREAM: rows are read past the caches.  Each is read once, so that those that do not fit the 256 MiB of the last of them only
// throw others out: 262144 rows of 1024 16-bit values 187 -> 160 us (5.1 TB/s), of which a lookup after it gives back 15; but 16384
// of 768, which are still there from what made them, 17 -> 22.
constexpr int kZeroRows = 16;
constexpr int64_t kStreamBytes = 256 << 20;
template <class T, int N, bool STREAM>
__global__ __launch_bounds__(256) void k_embed_sums(Sorted o, const T *grad, int64_t stride, int vocab, int dim, int chunk, int slices,
                                                    int64_t sum_waves, float scale, float *part, T *dw) {
    using P = Piece<T, N>;
    typedef float acc_t __attribute__((ext_vector_type(N)));
    const int lane = gs_lane();
    const int64_t w = (int64_t)blockIdx.x * 4 + gs_uniform((int)threadIdx.x >> 6);
    const auto put = [&](T *row, int d, acc_t x) {
        P y;
#pragma unroll
        for (int e = 0; e < N; e++) y.v[e] = (T)fmaf(x[e], scale, 0.f);  // no negative zeros from a negative scale
        if (d + N <= dim) *reinterpret_cast<P *>(row + d) = y;
        else
#pragma unroll
            for (int e = 0; e < N; e++)
                if (d + e < dim) row[d + e] = y.v[e];
    };
    if (w >= sum_waves) {
        const int64_t v0 = (w - sum_waves) * kZeroRows, v = v0 + lane;
        uint64_t none = __ballot(lane < kZeroRows && v < vocab && o.start[v] == o.start[v + 1]);
        for (; none; none &= none - 1) {
            T *row = dw + (v0 + __builtin_ctzll(none)) * dim;
            for (int d = lane * N; d < dim; d += 64 * N) put(row, d, acc_t{});
        }
        return;
    }
    const int64_t c = w / slices;
    const int d = (int)(w - c * slices) * 64 * N + lane * N;
    const int entries = o.start[vocab];
    const int64_t e0 = c * chunk;
    if (e0 >= entries) return;
    const int n = (int)min((int64_t)chunk, entries - e0);
    const bool from_before = e0 > 0 && o.id[e0 - 1] == o.id[e0], goes_on = e0 + n < entries && o.id[e0 + n - 1] == o.id[e0 + n];
    float *open = part + c * 2 * (int64_t)(slices * 64 * N);
    acc_t acc{};
    int cur = gs_uniform(o.id[e0]);
    bool first = true;
    const auto flush = [&](bool last) {
        const bool before = first && from_before;
        if (before || (last && goes_on)) {
            float *to = open + (before ? 0 : slices * 64 * N) + d;
#pragma unroll
            for (int e = 0; e < N; e++) to[e] = acc[e];
        } else {
            put(dw + (int64_t)cur * dim, d, acc);
        }
        first = false;
        acc = acc_t{};
    };
    constexpr int U = 8;
    for (int s = 0; s < n; s += 64) {
        const int64_t e = e0 + s + min(lane, n - s - 1);
        const int my_id = o.id[e];
        const uint32_t my_token = o.order[e];
        const int here = min(64, n - s);
        for (int k = 0; k < here; k += U) {
            typename P::vec x[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint32_t token = __builtin_amdgcn_readlane(my_token, min(k + u, here - 1));
                const T *row = grad + token * stride + d;
                if (d + N <= dim)
                    x[u] = STREAM ? __builtin_nontemporal_load(&reinterpret_cast<const P *>(row)->v) : reinterpret_cast<const P *>(row)->v;
                else
#pragma unroll
                    for (int q = 0; q < N; q++) x[u][q] = d + q < dim ? row[q] : (T)0;
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (k + u >= here) break;
                const int id = __builtin_amdgcn_readlane(my_id, k + u);
                if (id != cur) {
                    flush(false);
                    cur = id;
                }
#pragma unroll
                for (int q = 0; q < N; q++) acc[q] += (float)x[u][q];
            }
        }
    }
    flush(true);
}

// An id's parts together, in order: block c for the id whose entries start in chunk c and go on, a lane four columns, the waves
// equal runs of the parts, whose sums are added in order.  Most blocks find nothing: 262144 tokens 10 us.
template <class T>
__global__ __launch_bounds__(256) void k_embed_join(Sorted o, int vocab, int dim, int chunk, int64_t ld, float scale, const float *part, T *dw) {
    __shared__ f32x4 red[4][64];
    const int64_t c = blockIdx.x, e1 = (c + 1) * chunk;
    const int entries = o.start[vocab];
    if (e1 >= entries) return;
    const int id = o.id[e1];
    if (o.id[e1 - 1] != id || o.start[id] < c * chunk) return;
    const int64_t last = (o.start[id + 1] - 1) / chunk, parts = last - c + 1;
    const int lane = gs_lane(), wave = threadIdx.x >> 6, d = blockIdx.y * 256 + lane * 4;
    const int64_t a = parts * wave / 4, b = parts * (wave + 1) / 4;
    f32x4 x{0.f, 0.f, 0.f, 0.f};
    if (d < dim) {
#pragma unroll 8
        for (int64_t k = a; k < b; k++) x += *reinterpret_cast<const f32x4 *>(part + ((c + k) * 2 + (k == 0)) * ld + d);
    }
    red[wave][lane] = x;
    __syncthreads();
    if (wave > 0) return;
    for (int k = 1; k < 4; k++) x += red[k][lane];
    for (int e = 0; e < 4; e++)
        if (d + e < dim) dw[(int64_t)id * dim + d + e] = (T)fmaf(x[e], scale, 0.f);
}

// The whole gradient of at most 1024 tokens, for latency: a workgroup takes a range of ids, looks through all tokens for them
// (one each per thread), and writes the range's rows: zeros, a wave the sum of an id's tokens, all waves together that of an id with
// more than kLong of them.  What bounds it is dW, whose rows are mostly zeros: 512 tokens, 30522 rows of 384 fp32 values 14.8 us (47
// MB, 3.2 TB/s) against 42 in three launches.
constexpr int kFewTokens = 1024, kLong = 32;
template <class T, int N>
__global__ __launch_bounds__(1024) void k_embed_few(Tokens t, const T *grad, int64_t stride, int dim, float scale, T *dw) {
    using P = Piece<T, N>;
    typedef float acc_t __attribute__((ext_vector_type(N)));
    __shared__ int list[kFewTokens], sorted[kFewTokens], runs[kFewTokens + 1], wave_n[16];  // key << 10 | token
    __shared__ uint32_t has[128];
    __shared__ __align__(16) acc_t part[16][64];
    const int tid = threadIdx.x, lane = gs_lane(), wave = gs_uniform(tid >> 6);
    const int width = 1 << t.shift, id0 = blockIdx.x << t.shift, rows = min(width, t.vocab - id0);
    const int id = tid < t.n ? t.id(tid) : -1;
    const bool on = id >= 0 && id >> t.shift == (int)blockIdx.x;
    const auto place = [&](bool flag) {  // of this thread's among the flags, and how many there are
        const uint64_t m = __ballot(flag);
        __syncthreads();
        if (lane == 0) wave_n[wave] = __popcll(m);
        __syncthreads();
        int at = __popcll(m & gs_lanemask_lt()), all = 0;
        for (int w = 0; w < 16; w++) {
            if (w < wave) at += wave_n[w];
            all += wave_n[w];
        }
        return make_int2(at, all);
    };
    if (tid < 128) has[tid] = 0;
    const int2 mine = place(on);
    const int n = mine.y;
    if (on) {
        const int key = id - id0;
        list[mine.x] = key << 10 | tid;
        atomicOr(&has[key >> 5], 1u << (key & 31));
    }
    __syncthreads();
    const auto put = [&](int row, int d, acc_t x) {
        P y;
#pragma unroll
        for (int e = 0; e < N; e++) y.v[e] = (T)fmaf(x[e], scale, 0.f);  // no negative zeros from a negative scale
        T *to = dw + (int64_t)(id0 + row) * dim + d;
        if (d + N <= dim) *reinterpret_cast<P *>(to) = y;
        else
#pragma unroll
            for (int e = 0; e < N; e++)
                if (d + e < dim) to[e] = y.v[e];
    };
    for (int r = wave; r < rows; r += 16)
        if (!(has[r >> 5] >> (r & 31) & 1))
            for (int d = lane * N; d < dim; d += 64 * N) put(r, d, acc_t{});
    if (n == 0) return;
    // the keys differ, since they hold their token
    if (tid < n) {
        const int x = list[tid];
        int at = 0;
        for (int k = 0; k < n; k++) at += list[k] < x;
        sorted[at] = x;
    }
    __syncthreads();
    const bool starts = tid < n && (tid == 0 || sorted[tid] >> 10 != sorted[tid - 1] >> 10);
    const int2 run = place(starts);
    if (starts) runs[run.x] = tid;
    if (tid == 0) runs[run.y] = n;
    __syncthreads();
    // rows a to b of the sorted list
    const auto sum = [&](int a, int b, int d) {
        acc_t x{};
        constexpr int U = 8;
        for (int k = a; k < b; k += U) {
            typename P::vec v[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const T *row = grad + (sorted[min(k + u, b - 1)] & 1023) * stride + d;
                if (d + N <= dim) v[u] = reinterpret_cast<const P *>(row)->v;
                else
#pragma unroll
                    for (int e = 0; e < N; e++) v[u][e] = d + e < dim ? row[e] : (T)0;
            }
#pragma unroll
            for (int u = 0; u < U; u++)
                if (k + u < b) {
#pragma unroll
                    for (int e = 0; e < N; e++) x[e] += (float)v[u][e];
                }
        }
        return x;
    };
    const int slices = (dim + 64 * N - 1) / (64 * N);
    for (int w = wave; w < run.y * slices; w += 16) {
        const int r = w / slices, d = (w - r * slices) * 64 * N + lane * N;
        if (runs[r + 1] - runs[r] <= kLong) put(sorted[runs[r]] >> 10, d, sum(runs[r], runs[r + 1], d));
    }
    for (int r = 0; r < run.y; r++) {
        const int a = runs[r], len = runs[r + 1] - a;
        if (len <= kLong) continue;
        for (int s = 0; s < slices; s++) {
            const int d = s * 64 * N + lane * N;
            part[wave][lane] = sum(a + len * wave / 16, a + len * (wave + 1) / 16, d);
            __syncthreads();
            if (wave == 0) {
                acc_t x = part[0][lane];
                for (int k = 1; k < 16; k++) x += part[k][lane];
                put(sorted[a] >> 10, d, x);
            }
            __syncthreads();
        }
    }
}

// ---------------------------------------------------------------- host

int check_lookup(const gs_lookup *l) {
    GS_REQUIRE(l, "lookup is NULL");
    GS_REQUIRE(l->id_bytes == 4 || l->id_bytes == 8, "ids of %d bytes: 4 or 8", l->id_bytes);
    GS_REQUIRE(known(l->type) || l->type == GS_H_I8, "unknown weight type %d", l->type);
    GS_REQUIRE(l->tokens >= 0 && l->tokens <= (1 << 28), "%lld tokens outside [0, 2^28]", (long long)l->tokens);
    GS_REQUIRE(l->vocab >= 1 && l->vocab <= (1 << 20), "vocab=%d outside [1, 2^20]", l->vocab);
    GS_REQUIRE(l->dim >= 1 && l->dim <= 32768, "dim=%d outside [1, 32768]", l->dim);
    return GS_OK;
}

template <class T, class O, int N>
int run_lookup(const gs_lookup *l, const float *scales, O *out, hipStream_t s) {
    const int pieces = (l->dim + N - 1) / N;
    const int64_t total = l->tokens * pieces;
    const Ids ids{l->ids_d, l->id_bytes};
    constexpr int U = 4;
    const int64_t blocks = (total + 256 * U - 1) / (256 * U);
    GS_REQUIRE(blocks < (1ll << 24), "%lld tokens of %d values exceed a grid", (long long)l->tokens, l->dim);
#define GSV_EMBED(TAIL)                                                                                                            \
    hipLaunchKernelGGL((k_embed<T, O, N, U, TAIL>), dim3((unsigned)blocks), dim3(256), 0, s, ids, (const T *)l->weight_d,            \
                       l->weight_row_stride, scales, l->vocab, l->dim, (uint32_t)pieces, total, l->scale, out)
    if (l->dim % N) GSV_EMBED(true);
    else GSV_EMBED(false);
#undef GSV_EMBED
    GS_CHECK_LAUNCH();
    return GS_OK;
}

struct GradPlan {
    int shift, ranges, segs, chunk, slices, n_vec;
    bool few, split;
    int64_t seg_size, chunks, ld;
    Sorted o;
    uint32_t *pos;
    uint16_t *low;
    int *counts, *begin;
    float *part;
};
GradPlan plan_grad(gs_arena &a, const gs_lookup *l) {
    GradPlan p{};
    while ((kRanges << p.shift) < l->vocab) p.shift++;
    p.ranges = (l->vocab + (1 << p.shift) - 1) >> p.shift;
    p.few = l->tokens <= kFewTokens;
    p.split = l->tokens > order_waves(kDirectLds, p.shift) * kDirectWave;
    if (p.few) return p;
    p.seg_size = kSegTokens;
    while (p.seg_size * kSegs < l->tokens) p.seg_size *= 2;
    p.segs = (int)((l->tokens + p.seg_size - 1) / p.seg_size);
    p.chunk = 16;
    while (p.chunk < 128 && (int64_t)p.chunk * 1024 < l->tokens) p.chunk *= 2;
    p.chunks = (l->tokens + p.chunk - 1) / p.chunk;
    p.n_vec = l->type == GS_H_F32 ? 4 : 8;
    p.slices = (l->dim + 64 * p.n_vec - 1) / (64 * p.n_vec);
    p.ld = (int64_t)p.slices * 64 * p.n_vec;
    p.o.start = a.take<int>((size_t)l->vocab + 1);
    p.o.order = a.take<uint32_t>(l->tokens);
    p.o.id = a.take<int>(l->tokens);
    if (p.split) {
        p.pos = a.take<uint32_t>(l->tokens);
        p.low = a.take<uint16_t>(l->tokens);
        p.counts = a.take<int>((size_t)kRanges * p.segs);
        p.begin = a.take<int>((size_t)kRanges * p.segs);
    }
    p.part = a.take<float>((size_t)p.chunks * 2 * p.ld);
    return p;
}

template <class T, int N>
int run_grad(const gs_lookup *l, const GradPlan &p, const void *grad_d, int64_t stride, void *dweight_d, hipStream_t s) {
    const int64_t padding = l->padding >= 0 && l->padding < l->vocab ? l->padding : -1;
    const Tokens t{Ids{l->ids_d, l->id_bytes}, l->tokens, padding, l->vocab, p.shift, p.ranges};
    if (p.few) {
        hipLaunchKernelGGL((k_embed_few<T, N>), dim3(p.ranges), dim3(1024), 0, s, t, (const T *)grad_d, stride, l->dim, l->scale, (T *)dweight_d);
        GS_CHECK_LAUNCH();
        return GS_OK;
    }
    const int width = 1 << p.shift, waves = order_waves(p.split ? kOrderLds : kDirectLds, p.shift);
    const int lds = (waves + 1) * width * 4 + (p.split ? 0 : waves * kDirectWave * 4);
    static std::atomic<uint64_t> set{0}, set_split{0};
    if (p.split) {
        hipLaunchKernelGGL(k_split, dim3(p.segs), dim3(kSplitThreads), 0, s, t, p.seg_size, p.segs, p.pos, p.low, p.counts, p.begin);
        GS_CHECK_LAUNCH();
        if (int rc = allow_lds(reinterpret_cast<const void *>(&k_order<true>), kOrderMost, set_split)) return rc;
        hipLaunchKernelGGL(k_order<true>, dim3(p.ranges), dim3(1024), lds, s, t, p.seg_size, p.segs, p.pos, p.low, p.counts, p.begin, p.o);
    } else {
        if (int rc = allow_lds(reinterpret_cast<const void *>(&k_order<false>), kOrderMost, set)) return rc;
        hipLaunchKernelGGL(k_order<false>, dim3(p.ranges), dim3(1024), lds, s, t, p.seg_size, p.segs, p.pos, p.low, p.counts, p.begin, p.o);
    }
    GS_CHECK_LAUNCH();
    const int64_t sum_waves = (p.chunks * p.slices + 3) / 4 * 4, zero_waves = ((int64_t)l->vocab + kZeroRows - 1) / kZeroRows;
#define GSV_SUMS(STREAM)                                                                                                             \
    hipLaunchKernelGGL((k_embed_sums<T, N, STREAM>), dim3((unsigned)((sum_waves + zero_waves + 3) / 4)), dim3(256), 0, s, p.o,         \
                       (const T *)grad_d, stride, l->vocab, l->dim, p.chunk, p.slices, sum_waves, l->scale, p.part, (T *)dweight_d)
    if (l->tokens * l->dim * (int64_t)sizeof(T) > kStreamBytes) GSV_SUMS(true);
    else GSV_SUMS(false);
#undef GSV_SUMS
    GS_CHECK_LAUNCH();
    if (p.chunks > 1) {
        hipLaunchKernelGGL((k_embed_join<T>), dim3((unsigned)(p.chunks - 1), (l->dim + 255) / 256), dim3(256), 0, s, p.o, l->vocab, l->dim,
                           p.chunk, p.ld, l->scale, p.part, (T *)dweight_d);
        GS_CHECK_LAUNCH();
    }
    return GS_OK;
}

template <class T>
int run_float_lookup(const gs_lookup *l, void *out_d, hipStream_t s) {
    if (l->weight_dim_stride == 1) return run_lookup<T, T, 16 / sizeof(T)>(l, nullptr, (T *)out_d, s);
    const int64_t total = l->tokens * l->dim;
    hipLaunchKernelGGL((k_embed_strided<T>), dim3(gs_blocks(total, 256, 1 << 16)), dim3(256), 0, s, Ids{l->ids_d, l->id_bytes},
                       (const T *)l->weight_d, l->weight_row_stride, l->weight_dim_stride, l->vocab, l->dim, total, l->scale, (T *)out_d);
    GS_CHECK_LAUNCH();
    return GS_OK;
}

}  // namespace gsv

using namespace gsv;

extern "C" int gs_embed_tokens(const gs_lookup *l, void *out_d, void *stream) {
    if (int rc = check_lookup(l)) return rc;
    const bool q8 = l->type == GS_H_I8;
    GS_REQUIRE(known(l->out_type) && (q8 || l->out_type == l->type), "output type %d of a weight of type %d", l->out_type, l->type);
    GS_REQUIRE(!q8 || l->weight_dim_stride == 1, "8-bit rows with a stride between values");
    if (l->tokens == 0) return GS_OK;
    GS_REQUIRE(l->ids_d && l->weight_d && out_d && (!q8 || l->scales_d), "NULL ids, weight, scales or output");
    const hipStream_t s = gs_stream(stream);
    if (q8) {
        if (l->out_type == GS_H_F32) return run_lookup<int8_t, float, 4>(l, l->scales_d, (float *)out_d, s);
        if (l->out_type == GS_H_F16) return run_lookup<int8_t, _Float16, 8>(l, l->scales_d, (_Float16 *)out_d, s);
        return run_lookup<int8_t, __bf16, 8>(l, l->scales_d, (__bf16 *)out_d, s);
    }
    if (l->type == GS_H_F32) return run_float_lookup<float>(l, out_d, s);
    if (l->type == GS_H_F16) return run_float_lookup<_Float16>(l, out_d, s);
    return run_float_lookup<__bf16>(l, out_d, s);
}

extern "C" int gs_embed_tokens_grad_workspace(const gs_lookup *l, size_t *bytes) {
    if (int rc = check_lookup(l)) return rc;
    GS_REQUIRE(bytes, "NULL size pointer");
    gs_arena a{nullptr, 0, 0};
    plan_grad(a, l);
    *bytes = a.used;
    return GS_OK;
}

extern "C" int gs_embed_tokens_grad(const gs_lookup *l, const void *grad_d, int64_t grad_row_stride, void *dweight_d, void *workspace_d,
                                    size_t workspace_bytes, void *stream) {
    if (int rc = check_lookup(l)) return rc;
    GS_REQUIRE(l->type != GS_H_I8, "8-bit rows have no gradient");
    GS_REQUIRE(grad_row_stride >= 0, "negative stride of the gradient");
    gs_arena a{(char *)workspace_d, 0, workspace_bytes};
    const GradPlan p = plan_grad(a, l);
    if (!a.ok()) {
        gs_set_error("embed_tokens_grad workspace too small: need %zu bytes, got %zu", a.used, workspace_bytes);
        return GS_ENOSPC;
    }
    GS_REQUIRE((workspace_d || a.used == 0) && dweight_d && ((l->ids_d && grad_d) || l->tokens == 0), "NULL ids, gradient or workspace");
    const hipStream_t s = gs_stream(stream);
    if (l->type == GS_H_F32) return run_grad<float, 4>(l, p, grad_d, grad_row_stride, dweight_d, s);
    if (l->type == GS_H_F16) return run_grad<_Float16, 8>(l, p, grad_d, grad_row_stride, dweight_d, s);
    return run_grad<__bf16, 8>(l, p, grad_d, grad_row_stride, dweight_d, s);
}
