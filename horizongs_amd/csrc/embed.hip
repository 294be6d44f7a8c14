// K18: embedding lookup with scaling, and its gradient by sorted ids (the per-camera appearance
// rows of the reference, scene/embedding.py:50-79, and any other table of learned rows).
//
//   out[i, :] = scale * W[ids[i], :]                       (zeros where ids[i] is no row of W)
//   dW[v, :]  = scale * sum over i with ids[i] = v of g[i, :]
//
// The lookup is a gather, bound by memory: one 16-byte piece of a row per lane.  500k rows of 32 floats
// 21.0 us (130 MB, 6.2 TB/s), 16k rows of 2048 bf16 16.3 us (5.7 TB/s).
//
// The gradient is summed in a fixed order, without float atomics, so it is the same bits on every
// run.  In its general form the (id, i) pairs are sorted by id (stable), the sorted list is cut into
// equal pieces -- not into rows, so a row named by half of the entries costs no more than any other --
// and each piece sums its runs in f32.  Runs inside a piece are written at once; the pieces' first and
// last runs are joined through LDS inside a workgroup and through a workspace between workgroups.
// Forms, by the number of ids n, of rows V and the columns per lane (bwd_plan):
//   n <= 1,024               one launch, a workgroup per id                       (600 x 2048: 9 us)
//   V * columns <= 128       tables of sums in LDS, no sort     (500k x 32 f32, 16 rows: 20 us)
//   n <= 24,576 (16,384 if V < 2048)
//                            sorted by ranges of ids, one launch   (16k x 2048 bf16, 65,536 rows: 68 us)
//   more                     radix sort           (500k x 32 f32 into a million rows: 52 us in order, 76 in any)
// Times what the same bytes take as a large copy (5 TB/s): ids sorted by ranges 1.0, many ids in order 1.3, few
// rows 1.4, the radix sort of ids in any order 1.9 (a million rows) to 3 (404 rows: 41 us, of which 20 are the sort's
// three launches and 16 the sums).
#include "rows.h"

namespace hgsr {

// ------------------------------------------------------------------------------------- lookup

template <typename WT, typename OT, typename I, int VEC, bool STREAM>
__global__ __launch_bounds__(256) void embed_fwd_kernel(uint32_t chunks, FastDiv per_row, uint32_t V, uint32_t D,
                                                        const WT* __restrict__ w, int64_t wstride, RowIds<I> ids,
                                                        int64_t row0, float scale, OT* __restrict__ out) {
    const uint32_t c = blockIdx.x * 256 + threadIdx.x;
    if (c >= chunks) return;
    const uint32_t r = per_row.div(c), col = min((c - r * per_row.d) * VEC, D - VEC);  // rows end on a whole piece
    const uint32_t id = ids.get(row0 + r, V);
    Vec<OT, VEC> o;
    if (id < V) {
        const Vec<WT, VEC> x = load_vec<WT, VEC>(w + (int64_t)id * wstride + col);
#pragma unroll
        for (int k = 0; k < VEC; ++k) o.v[k] = (OT)((float)x.v[k] * scale);
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) o.v[k] = (OT)0.0f;
    }
    OT* to = out + (row0 + r) * (int64_t)D + col;
    if (STREAM)
        stream_vec<OT, VEC>(to, o);
    else
        store_vec<OT, VEC>(to, o);
}

// --------------------------------------------------------------------------- zeros of the table
// A dense gradient's zeros are stored by extra workgroups of the launches that sort the ids: the
// sort is a chain of short, latency-bound kernels, and the memory is free meanwhile.  Rows that an
// id names are stored again by the sums.
struct ZeroPart {
    uint4* p;        // whole 16-byte units
    int64_t units;
    uint16_t* edge[2];  // what lies before the first and behind the last unit
    int nedge[2];
};
constexpr int kZeroUnits = 2048;  // per workgroup and turn: 32 KB
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// workgroup `block` of `blocks`; the zeros go past the caches (16k x 2048 bf16 ids into 65,536 rows:
// 89 us, 100 us with cached stores, which the sums' reads then have to push out)
template <int THREADS>
__device__ __forceinline__ void store_zeros(const ZeroPart& z, int64_t block, int64_t blocks) {
    for (int64_t u0 = block * kZeroUnits + threadIdx.x; u0 < z.units; u0 += blocks * kZeroUnits) {
#pragma unroll
        for (int k = 0; k < kZeroUnits / THREADS; ++k)
            if (u0 + k * THREADS < z.units)
                __builtin_nontemporal_store(u32x4{0, 0, 0, 0}, reinterpret_cast<u32x4*>(z.p) + u0 + k * THREADS);
    }
    if (block == 0 && threadIdx.x < 8) {
        if ((int)threadIdx.x < z.nedge[0]) z.edge[0][threadIdx.x] = 0;
        if ((int)threadIdx.x < z.nedge[1]) z.edge[1][threadIdx.x] = 0;
    }
}

__global__ __launch_bounds__(256) void zero_kernel(ZeroPart z) { store_zeros<256>(z, blockIdx.x, gridDim.x); }

// ------------------------------------------------------------------------------ sort of (id, i)
// Both forms are radix sorts, least significant digit first.  An entry's place among its wave's
// entries of one digit: `match` of the lanes that hold the digit, one ballot per bit; the first of
// them adds their number to the wave's count of the digit.
template <int MOST>
__device__ __forceinline__ uint64_t match(uint32_t d, bool on, int bits) {
    uint64_t same = __ballot(on);
    if (!on) same = ~same;
#pragma unroll
    for (int k = 0; k < MOST; ++k)
        if (k < bits) {
            const uint64_t m = __ballot((d >> k) & 1);
            same &= (d >> k) & 1 ? m : ~m;
        }
    return same;
}
__device__ __forceinline__ uint64_t below(int lane) { return (1ull << lane) - 1; }

__device__ __forceinline__ uint32_t wave_scan(uint32_t v, int lane) {  // inclusive
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

// Up to 24,576 entries: one launch.  The ids are cut into up to 256 ranges, a workgroup each: it
// reads all ids, keeps the positions of its own in LDS (in order) and counts the smaller ones, which
// is where its part of the list starts; then it sorts what it kept by the ids' remaining bits.  A
// range that does not fit (an id that half of the entries name) is sorted in global memory.
// (One workgroup for all: 42 us at 16,384 entries, LDS-bound; counting, for each entry, the ones
// before it: 36 us of the whole chip; this: 14.)
// Up to where: 24,000 ids of 65,536 rows of 64 floats 25 us if they are spread evenly, 46 if the low ones are
// frequent (Zipf), by the radix sort's two passes 40 and 41; 32,000 ids 36 and 57, 40 and 42.  Up to 2,047
// rows that sort has one pass: 24,000 of 404 rows 25 us by either, 48 and 26 if half of the ids are one;
// 10,000 of 404 17 and 24, 22 and 26.
constexpr int kBucketMost = 24576, kBucketMostOfOne = 16384;
constexpr int kBucketKeep = 8192;  // positions that a workgroup keeps
constexpr int kBucketRounds = kBucketKeep / 1024;
constexpr int kBucketLog = 8;
constexpr int kBucketBits = 9;   // per pass
constexpr int kCountMost = 512;  // entries that a workgroup sorts by counting

template <typename I>
struct BucketArgs {
    uint32_t n, V;
    RowIds<I> ids;
    int shift, passes, bits;
    uint32_t buckets;
    uint2 *out, *tmp;
};

// per wave and digit: counts -> where the wave's entries of the digit go (after all smaller digits and the
// earlier waves'); 1024 threads
__device__ __forceinline__ void digit_places(uint32_t (*cnt)[1 << kBucketBits], uint32_t* wsum, uint32_t bins) {
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
    uint32_t c[16], sum = 0;
    if ((uint32_t)tid < bins) {
#pragma unroll
        for (int q = 0; q < 16; ++q) c[q] = cnt[q][tid];
#pragma unroll
        for (int q = 0; q < 16; ++q) sum += c[q];
    }
    const uint32_t inc = wave_scan(sum, lane);
    if (lane == 63) wsum[w] = inc;
    __syncthreads();
    uint32_t to = inc - sum;
    for (int q = 0; q < w; ++q) to += wsum[q];
    if ((uint32_t)tid < bins) {
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            cnt[q][tid] = to;
            to += c[q];
        }
    }
    __syncthreads();
}

// the wave's next entries that hold digit d: their places, one after the other
__device__ __forceinline__ uint32_t take_places(uint32_t* cnt, uint32_t d, bool on, int bits, int lane) {
    const uint64_t same = match<kBucketBits>(d, on, bits);
    const int first = __ffsll((unsigned long long)same) - 1;
    uint32_t old = 0;
    if (on && lane == first) old = atomicAdd(&cnt[d], (uint32_t)__popcll(same));
    return __shfl(old, first) + __popcll(same & below(lane));
}

template <typename I>
__global__ __launch_bounds__(1024) void sort_bucket_kernel(const BucketArgs<I> a, ZeroPart zeros) {
    __shared__ uint16_t pos[kBucketKeep];
    __shared__ __align__(16) uint32_t cnt[16][1 << kBucketBits];
    __shared__ uint32_t wsum[2][16];
    if (blockIdx.x >= a.buckets) return store_zeros<1024>(zeros, blockIdx.x - a.buckets, gridDim.x - a.buckets);
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
    const uint32_t bucket = blockIdx.x, n = a.n, bins = 1u << a.bits;
    uint32_t m = 0, start = 0;
    for (uint32_t j0 = 0; j0 < n; j0 += kBucketKeep) {  // a wave's entries are consecutive
        const int rounds = (int)((min(n - j0, (uint32_t)kBucketKeep) + 1023) / 1024);
        const uint32_t base = j0 + w * rounds * 64 + lane;
        uint32_t k[kBucketRounds], mine = 0, less = 0;
#pragma unroll
        for (int r = 0; r < kBucketRounds; ++r)
            if (r < rounds) k[r] = base + r * 64 < n ? a.ids.get(base + r * 64, a.V) : ~0u;
#pragma unroll
        for (int r = 0; r < kBucketRounds; ++r)
            if (r < rounds) {
                mine += __popcll(__ballot(k[r] >> a.shift == bucket && k[r] != ~0u));
                less += __popcll(__ballot(k[r] >> a.shift < bucket));
            }
        if (lane == 0) {
            wsum[0][w] = mine;
            wsum[1][w] = less;
        }
        __syncthreads();
        uint32_t at = m;
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            if (q < w) at += wsum[0][q];
            m += wsum[0][q];
            start += wsum[1][q];
        }
#pragma unroll
        for (int r = 0; r < kBucketRounds; ++r)
            if (r < rounds) {
                const bool in = k[r] >> a.shift == bucket && k[r] != ~0u;
                const uint64_t b = __ballot(in);
                const uint32_t to = at + __popcll(b & below(lane));
                if (in && to < kBucketKeep) pos[to] = (uint16_t)(base + r * 64);
                at += __popcll(b);
            }
        __syncthreads();
    }
    if (m == 0) return;
    uint2 *out = a.out + start, *tmp = a.tmp + start;
    if (m > kBucketKeep) {
        // the range once more, its entries into global memory in order: done if they are one id's
        uint2* src = a.passes & 1 ? tmp : out;
        uint32_t filled = 0, lowest = ~0u, highest = 0;
        for (uint32_t j0 = 0; j0 < n; j0 += kBucketKeep) {
            const uint32_t base = j0 + w * kBucketRounds * 64 + lane;
            uint32_t k[kBucketRounds], mine = 0;
#pragma unroll
            for (int r = 0; r < kBucketRounds; ++r) k[r] = base + r * 64 < n ? a.ids.get(base + r * 64, a.V) : ~0u;
#pragma unroll
            for (int r = 0; r < kBucketRounds; ++r)
                mine += __popcll(__ballot(k[r] >> a.shift == bucket && k[r] != ~0u));
            if (lane == 0) wsum[0][w] = mine;
            __syncthreads();
            uint32_t at = filled;
#pragma unroll
            for (int q = 0; q < 16; ++q) {
                if (q < w) at += wsum[0][q];
                filled += wsum[0][q];
            }
#pragma unroll
            for (int r = 0; r < kBucketRounds; ++r) {
                const bool in = k[r] >> a.shift == bucket && k[r] != ~0u;
                const uint64_t b = __ballot(in);
                if (in) {
                    src[at + __popcll(b & below(lane))] = make_uint2(k[r], base + r * 64);
                    lowest = min(lowest, k[r]);
                    highest = max(highest, k[r]);
                }
                at += __popcll(b);
            }
            __syncthreads();
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            lowest = min(lowest, (uint32_t)__shfl_xor((int)lowest, d));
            highest = max(highest, (uint32_t)__shfl_xor((int)highest, d));
        }
        if (lane == 0) {
            wsum[0][w] = lowest;
            wsum[1][w] = highest;
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            lowest = min(lowest, wsum[0][q]);
            highest = max(highest, wsum[1][q]);
        }
        __syncthreads();
        const uint32_t share = (m + 1023) / 1024 * 64, i0 = w * share, i1 = min(m, i0 + share);
        if (lowest == highest) {
            if (src == tmp)
                for (uint32_t i = tid; i < m; i += 1024) out[i] = tmp[i];
            return;
        }
        for (int pass = 0; pass < a.passes; ++pass) {
            const int sh = pass * a.bits;
            uint2* dst = src == out ? tmp : out;
            for (uint32_t b = tid; b < 16 * bins; b += 1024) cnt[b >> a.bits][b & (bins - 1)] = 0;
            __syncthreads();
#pragma unroll 8
            for (uint32_t i = i0 + lane; i < i1; i += 64) atomicAdd(&cnt[w][(src[i].x >> sh) & (bins - 1)], 1u);
            __syncthreads();
            digit_places(cnt, wsum[0], bins);
            for (uint32_t i = i0; i < i1; i += 4 * 64) {
                uint2 e[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) e[r] = src[min(i + r * 64 + lane, i1 - 1)];
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (i + r * 64 < i1) {
                        const bool on = i + r * 64 + lane < i1;
                        const uint32_t to = take_places(cnt[w], (e[r].x >> sh) & (bins - 1), on, a.bits, lane);
                        if (on) dst[to] = e[r];
                    }
            }
            __syncthreads();
            src = dst;
        }
        return;
    }
    const int rounds = (m + 1023) / 1024;
    const uint32_t base = w * rounds * 64 + lane;
    if (a.passes == 0) {  // a range of one id
        for (int r = 0; r < rounds; ++r)
            if (base + r * 64 < m) out[base + r * 64] = make_uint2(bucket, pos[base + r * 64]);
        return;
    }
    if (m <= kCountMost) {
        // few: an entry's place is the number of entries before it, each comparing with all; `parts`
        // threads share an entry's comparisons
        uint32_t *id = cnt[0], *before = cnt[0] + kCountMost;
        const uint32_t width = m <= 64 ? 64 : m <= 128 ? 128 : m <= 256 ? 256 : 512, parts = 1024 / width;
        if ((uint32_t)tid < width) {
            id[tid] = (uint32_t)tid < m ? a.ids.get(pos[tid], a.V) : ~0u;
            before[tid] = 0;
        }
        __syncthreads();
        const uint32_t i = tid & (width - 1), own = id[i], share = width / parts, j0 = (tid / width) * share;
        uint32_t sum = 0;
        for (uint32_t j = j0; j < j0 + share; j += 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(id + j);
            sum += v.x < own + (j < i);
            sum += v.y < own + (j + 1 < i);
            sum += v.z < own + (j + 2 < i);
            sum += v.w < own + (j + 3 < i);
        }
        if (i < m) atomicAdd(&before[i], sum);
        __syncthreads();
        if ((uint32_t)tid < m) out[before[tid]] = make_uint2(own, pos[tid]);
        return;
    }
    uint32_t k[kBucketRounds], place[kBucketRounds];
    uint16_t p[kBucketRounds];
    for (int pass = 0; pass < a.passes; ++pass) {
        const int sh = pass * a.bits;
#pragma unroll
        for (int r = 0; r < kBucketRounds; ++r)
            if (r < rounds) {
                p[r] = base + r * 64 < m ? pos[base + r * 64] : 0;
                k[r] = a.ids.get(p[r], a.V);
            }
        for (uint32_t b = tid; b < 16 * bins; b += 1024) cnt[b >> a.bits][b & (bins - 1)] = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kBucketRounds; ++r)
            if (r < rounds)
                place[r] = take_places(cnt[w], (k[r] >> sh) & (bins - 1), base + r * 64 < m, a.bits, lane);
        __syncthreads();
        digit_places(cnt, wsum[0], bins);
#pragma unroll
        for (int r = 0; r < kBucketRounds; ++r)
            if (r < rounds && base + r * 64 < m) {
                const uint32_t to = cnt[w][(k[r] >> sh) & (bins - 1)] + place[r];
                if (pass == a.passes - 1)
                    out[to] = make_uint2(k[r], p[r]);
                else
                    pos[to] = p[r];
            }
        __syncthreads();
    }
}

// More: digits of up to 11 bits, per pass three launches: the tiles' digit counts, their prefix over
// the tiles, a stable scatter.  The first pass also notes whether the ids ascend already (a compacted
// index does): the rest of the sort then ends at once, and the sums read the ids themselves.
constexpr int kSortRounds = 8;
constexpr int kSortTile = 256 * kSortRounds;  // entries per workgroup: 4 waves x 8 rounds x 64 lanes
constexpr int kSortBits = 11;

template <typename I>
struct SortArgs {
    uint32_t n, V;
    RowIds<I> ids;
    const uint2* in;   // nullptr: the first pass, entries from the ids
    uint2* out;
    int shift, bits;
    uint32_t tiles;
    uint32_t* hist;    // [tiles][1 << bits]
    uint32_t* total;   // [1 << bits]
    uint32_t* ascend;  // [1 + tiles]: the verdict, then the tiles' own
};

template <bool FIRST, typename I>
__device__ __forceinline__ uint2 sort_entry(const SortArgs<I>& a, uint32_t i) {
    if (FIRST) return make_uint2(a.ids.get(i, a.V), i);
    return a.in[i];
}

template <bool FIRST, typename I>
__global__ __launch_bounds__(256) void sort_count_kernel(const SortArgs<I> a, ZeroPart zeros) {
    __shared__ uint32_t h[1 << kSortBits];
    __shared__ uint32_t id[FIRST ? kSortTile + 1 : 1];
    if (!FIRST && *a.ascend) return;
    if (blockIdx.x >= a.tiles) return store_zeros<256>(zeros, blockIdx.x - a.tiles, gridDim.x - a.tiles);
    const uint32_t bins = 1u << a.bits, base = blockIdx.x * kSortTile;
    uint32_t v[kSortRounds];
#pragma unroll
    for (int k = 0; k < kSortRounds; ++k) {
        const uint32_t i = base + k * 256 + threadIdx.x;
        v[k] = i < a.n ? sort_entry<FIRST>(a, i).x : ~0u;
    }
    if (FIRST && threadIdx.x == 0) id[kSortTile] = base + kSortTile < a.n ? a.ids.get(base + kSortTile, a.V) : ~0u;
    for (uint32_t b = threadIdx.x; b < bins; b += 256) h[b] = 0;
    if (FIRST) {
#pragma unroll
        for (int k = 0; k < kSortRounds; ++k) id[k * 256 + threadIdx.x] = v[k];
    }
    __syncthreads();
    int up = 1;
#pragma unroll
    for (int k = 0; k < kSortRounds; ++k)
        if (v[k] != ~0u) {
            atomicAdd(&h[(v[k] >> a.shift) & (bins - 1)], 1u);
            if (FIRST) up &= v[k] <= id[k * 256 + threadIdx.x + 1];
        }
    up = __syncthreads_and(up);
    if (FIRST && threadIdx.x == 0) a.ascend[1 + blockIdx.x] = up;
    for (uint32_t b = threadIdx.x; b < bins; b += 256) a.hist[(size_t)blockIdx.x * bins + b] = h[b];
}

// 64 digits per workgroup, a share of the tiles per wave: exclusive prefix of each digit's counts
// over the tiles, and its total.  The last workgroup of the first pass joins the tiles' verdicts.
template <bool FIRST, typename I>
__global__ __launch_bounds__(1024) void sort_scan_kernel(const SortArgs<I> a) {
    __shared__ uint32_t part[16][64];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const uint32_t bins = 1u << a.bits, bin = blockIdx.x * 64 + lane;
    if (FIRST && blockIdx.x == gridDim.x - 1) {
        int up = 1;
        for (uint32_t t = threadIdx.x; t < a.tiles; t += 1024) up &= a.ascend[1 + t];
        up = __syncthreads_and(up);
        if (threadIdx.x == 0) a.ascend[0] = up;
        return;
    }
    if (!FIRST && *a.ascend) return;
    uint32_t carry = 0;
    for (uint32_t t0 = 0; t0 < a.tiles; t0 += 256) {
        uint32_t v[16], sum = 0;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const uint32_t t = t0 + w * 16 + k;
            v[k] = t < a.tiles && bin < bins ? a.hist[(size_t)t * bins + bin] : 0;
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) sum += v[k];
        part[w][lane] = sum;
        __syncthreads();
        uint32_t at = carry;
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            const uint32_t p = part[q][lane];
            if (q < w) at += p;
            carry += p;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const uint32_t t = t0 + w * 16 + k;
            if (t < a.tiles && bin < bins) a.hist[(size_t)t * bins + bin] = at;
            at += v[k];
        }
    }
    if (w == 0 && bin < bins) a.total[bin] = carry;
}

template <bool FIRST, typename I>
__global__ __launch_bounds__(256) void sort_scatter_kernel(const SortArgs<I> a, ZeroPart zeros) {
    __shared__ uint32_t cnt[4][1 << kSortBits];  // per wave: count, then where its entries of the digit go
    __shared__ uint32_t wsum[4];
    if (*a.ascend) return;
    if (blockIdx.x >= a.tiles) return store_zeros<256>(zeros, blockIdx.x - a.tiles, gridDim.x - a.tiles);
    const uint32_t bins = 1u << a.bits;
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
    const uint32_t base = blockIdx.x * kSortTile + w * (kSortTile / 4);
    uint2 e[kSortRounds];
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
        const uint32_t i = base + r * 64 + lane;
        e[r] = i < a.n ? sort_entry<FIRST>(a, i) : make_uint2(0, 0);
    }
    // digits tid * PER .. of this tile start at (entries of smaller digits) + (theirs in earlier tiles)
    constexpr int PER = (1 << kSortBits) / 256;
    uint32_t mine[PER], off[PER], sum = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const uint32_t b = tid * PER + k;
        mine[k] = b < bins ? a.total[b] : 0;
        off[k] = b < bins ? a.hist[(size_t)blockIdx.x * bins + b] : 0;
        sum += mine[k];
    }
    for (uint32_t b = tid; b < 4 * bins; b += 256) cnt[b >> a.bits][b & (bins - 1)] = 0;
    __syncthreads();
    uint64_t same[kSortRounds];
    uint32_t old[kSortRounds];
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
        const bool on = base + r * 64 + lane < a.n;
        const uint32_t d = (e[r].x >> a.shift) & (bins - 1);
        same[r] = match<kSortBits>(d, on, a.bits);
        old[r] = 0;
        if (on && (same[r] & below(lane)) == 0) old[r] = atomicAdd(&cnt[w][d], (uint32_t)__popcll(same[r]));
    }
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r)
        old[r] = __shfl(old[r], __ffsll((unsigned long long)same[r]) - 1) + __popcll(same[r] & below(lane));
    const uint32_t inc = wave_scan(sum, lane);
    if (lane == 63) wsum[w] = inc;
    __syncthreads();
    uint32_t at = inc - sum;
    for (int k = 0; k < w; ++k) at += wsum[k];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const uint32_t b = tid * PER + k;
        if (b < bins) {
            uint32_t p = at + off[k];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint32_t c = cnt[q][b];
                cnt[q][b] = p;
                p += c;
            }
        }
        at += mine[k];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r)
        if (base + r * 64 + lane < a.n) a.out[cnt[w][(e[r].x >> a.shift) & (bins - 1)] + old[r]] = e[r];
}

// --------------------------------------------------------------------------------------- sums
// A subgroup of `lanes` lanes holds VEC columns per lane; columns beyond lanes * VEC: grid.y.
template <typename I>
struct SumArgs {
    uint32_t n, V;
    int64_t D;
    RowIds<I> ids;
    const uint2* list;       // sorted (id, i)
    const uint32_t* ascend;  // not null and set: the ids ascend by themselves, no list was made
    const void* g;
    int64_t gstride;
    void* dw;
    int64_t dwstride;
    int accumulate;
    float scale;
    int lanes;           // lanes per subgroup, a power of two
    int run;             // entries per subgroup
    uint32_t blocks;     // workgroups over the entries
    float *head, *tail;  // [blocks][D]: the sums of a workgroup's runs that began before it / go on after it
    uint32_t rows;       // table form: entries per workgroup; others: rows per zeroing workgroup
    uint8_t* named;      // table form: [blocks][V]
};

// The columns of a lane.  A row whose length no VEC divides ends on a whole piece all the same: its last
// lane's columns start before the piece (`skip` of them are the previous lane's too, and get the same
// values from both, except where something is added to them).
template <int VEC>
struct Cols {
    int64_t col;
    int skip;
    bool on;
    __device__ __forceinline__ Cols(int64_t D, int lanes, int ln, uint32_t slab) {
        const int64_t c = ((int64_t)slab * lanes + ln) * VEC;
        on = c < D;
        col = c < D - VEC ? c : D - VEC;
        skip = on ? (int)(c - col) : 0;
    }
};

template <typename OT, int VEC, bool STREAM = false, typename I>
__device__ __forceinline__ void put_row(const SumArgs<I>& a, uint32_t v, const Cols<VEC>& c, const float* acc) {
    OT* p = static_cast<OT*>(a.dw) + (int64_t)v * a.dwstride + c.col;
    Vec<OT, VEC> o;
    if (a.accumulate && c.skip) {
#pragma unroll
        for (int k = 1; k < VEC; ++k)
            if (k >= c.skip) p[k] = (OT)((float)p[k] + acc[k] * a.scale);
        return;
    }
    if (a.accumulate) {
        o = load_vec<OT, VEC>(p);
#pragma unroll
        for (int k = 0; k < VEC; ++k) o.v[k] = (OT)((float)o.v[k] + acc[k] * a.scale);
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) o.v[k] = (OT)(acc[k] * a.scale);
    }
    if (STREAM)
        stream_vec<OT, VEC>(p, o);
    else
        store_vec<OT, VEC>(p, o);
}

// a row that no id names: zeros whatever the scale
template <typename OT, int VEC, bool STREAM = false, typename I>
__device__ __forceinline__ void put_zeros(const SumArgs<I>& a, uint32_t v, const Cols<VEC>& c) {
    OT* p = static_cast<OT*>(a.dw) + (int64_t)v * a.dwstride + c.col;
    Vec<OT, VEC> o;
#pragma unroll
    for (int k = 0; k < VEC; ++k) o.v[k] = (OT)0.0f;
    if (STREAM)
        stream_vec<OT, VEC>(p, o);
    else
        store_vec<OT, VEC>(p, o);
}

template <typename T, int VEC>
__device__ __forceinline__ void add_vec(float* acc, const Vec<T, VEC>& x) {
#pragma unroll
    for (int c = 0; c < VEC; ++c) acc[c] += (float)x.v[c];
}

// acc of the first `live` subgroups (at least 1; the others hold nothing) summed into subgroup 0's, in
// a fixed tree; every thread of the workgroup calls it
template <int VEC>
__device__ __forceinline__ void sum_subgroups(Vec<float, VEC>* part, float* acc, int lanes, int live) {
    const int tid = threadIdx.x, s = tid / lanes;
    int h = 1;
    while (h < live) h <<= 1;
    for (h >>= 1; h > 0; h >>= 1) {
        if (s >= h && s < 2 * h) {
#pragma unroll
            for (int c = 0; c < VEC; ++c) part[tid].v[c] = acc[c];
        }
        __syncthreads();
        if (s < h) add_vec<float, VEC>(acc, part[tid + h * lanes]);
    }
}

// ---- few entries: one launch, a workgroup per entry.  The first of the entries that name a row
// sums them all (each subgroup every NS-th of them, joined through LDS); other workgroups store the
// zeros of the rows that no id names.  1,000 rows of 2048 bf16: 12 us, 16 by the sort; 25 if they are all
// one row's (72 with a comparison around each of the eight loads, which then wait for one another).
constexpr int kFewMost = 1024;
constexpr int kFewRows = 1024;  // rows per zeroing workgroup, at most

template <typename GT, typename OT, typename I, int VEC>
__global__ __launch_bounds__(256) void embed_few_kernel(const SumArgs<I> a) {
    constexpr int PER = kFewMost / 256;
    __shared__ Vec<float, VEC> part[256];
    __shared__ uint16_t match[kFewMost];
    __shared__ uint32_t count[PER][4];
    __shared__ uint8_t named[kFewRows];
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
    const int L = a.lanes, s = tid / L, ln = tid & (L - 1), NS = 256 / L;
    const Cols<VEC> c(a.D, L, ln, blockIdx.y);
    const int64_t col = c.col;
    const bool on = c.on;
    uint32_t mine[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) mine[k] = k * 256 + tid < (int)a.n ? a.ids.get(k * 256 + tid, a.V) : a.V;
    if (blockIdx.x >= a.n) {
        const uint32_t r0 = (blockIdx.x - a.n) * a.rows;
        for (uint32_t k = tid; k < a.rows; k += 256) named[k] = 0;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < PER; ++k)
            if (mine[k] < a.V && mine[k] >= r0 && mine[k] - r0 < a.rows) named[mine[k] - r0] = 1;
        __syncthreads();
        for (uint32_t k = s; k < a.rows && r0 + k < a.V; k += NS)
            if (on && !named[k]) put_zeros<OT, VEC>(a, r0 + k, c);
        return;
    }
    const uint32_t v = a.ids.get(blockIdx.x, a.V);
    if (v >= a.V) return;
    uint64_t same[PER];
    int earlier = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        same[k] = __ballot(mine[k] == v);
        earlier |= mine[k] == v && k * 256 + tid < (int)blockIdx.x;
        if (lane == 0) count[k][w] = __popcll(same[k]);
    }
    if (__syncthreads_or(earlier)) return;
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (q == w && mine[k] == v) match[m + __popcll(same[k] & below(lane))] = (uint16_t)(k * 256 + tid);
            m += count[k][q];
        }
    __syncthreads();
    float acc[VEC] = {};
    if (on) {
        const GT* g = static_cast<const GT*>(a.g) + col;
        uint32_t j = s;
        for (; j + 7 * NS < m; j += 8 * NS) {
            Vec<GT, VEC> x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] = load_vec<GT, VEC>(g + (int64_t)match[j + u * NS] * a.gstride);
#pragma unroll
            for (int u = 0; u < 8; ++u) add_vec<GT, VEC>(acc, x[u]);
        }
#pragma unroll 4
        for (; j < m; j += NS) add_vec<GT, VEC>(acc, load_vec<GT, VEC>(g + (int64_t)match[j] * a.gstride));
    }
    sum_subgroups<VEC>(part, acc, L, m < (uint32_t)NS ? (int)m : NS);
    if (s == 0 && on) put_row<OT, VEC>(a, v, c, acc);
}

// ---- few rows: no sort.  Every subgroup keeps a table of sums in LDS, its own, so a workgroup's
// entries are read once and in order; the subgroups' and then the workgroups' tables are added.
// 500k ids of rows of 32 floats: 16 rows 20.0 us (sorted: 37.8), 32 rows 24.0 (sorted: 37.6).
constexpr int kTableMost = 128;  // V * VEC: 128 KB of LDS
// Rows that a subgroup reads at once: the tables leave room for one or two workgroups per unit, so each has
// to keep many loads in flight.  500k ids, 20 rows of 64 floats: 8 / 12 / 16 / 24 rows 52 / 44 / 43 / 52 us;
// 16 rows of 16 bf16: 24 / 19 / 18.7 / 24.
constexpr int kTableRounds = 16;

template <typename GT, typename I, int VEC>
__global__ __launch_bounds__(256) void embed_table_kernel(const SumArgs<I> a) {
    extern __shared__ __align__(16) char smem[];
    Vec<float, VEC>* tab = reinterpret_cast<Vec<float, VEC>*>(smem);  // [V][256]
    __shared__ uint8_t named[kTableMost];
    const int tid = threadIdx.x, L = a.lanes, s = tid / L, ln = tid & (L - 1), NS = 256 / L;
    const Cols<VEC> c(a.D, L, ln, blockIdx.y);
    const int64_t col = c.col;
    const bool on = c.on;
    Vec<float, VEC> zero;
#pragma unroll
    for (int c = 0; c < VEC; ++c) zero.v[c] = 0.0f;
    for (uint32_t v = 0; v < a.V; ++v) tab[v * 256 + tid] = zero;
    if (tid < kTableMost) named[tid] = 0;
    __syncthreads();
    const GT* g = static_cast<const GT*>(a.g) + col;
    const uint64_t i1 = min((uint64_t)a.n, ((uint64_t)blockIdx.x + 1) * a.rows);
    for (uint64_t i0 = (uint64_t)blockIdx.x * a.rows + s; i0 < i1; i0 += kTableRounds * NS) {
        uint32_t id[kTableRounds];
        Vec<GT, VEC> x[kTableRounds];
#pragma unroll
        for (int u = 0; u < kTableRounds; ++u) {
            const int64_t i = i0 + u * NS;
            const int64_t j = i < (int64_t)i1 ? i : i1 - 1;
            id[u] = a.ids.get(j, a.V);
            if (j != i) id[u] = a.V;
            x[u] = load_vec<GT, VEC>(g + j * a.gstride);
        }
#pragma unroll
        for (int u = 0; u < kTableRounds; ++u)
            if (id[u] < a.V) {
                Vec<float, VEC> t = tab[id[u] * 256 + tid];
                add_vec<GT, VEC>(t.v, x[u]);
                tab[id[u] * 256 + tid] = t;
                if (ln == 0) named[id[u]] = 1;
            }
    }
    __syncthreads();
    for (uint32_t v = s; v < a.V; v += NS) {
        float acc[VEC] = {};
        for (int q = 0; q < NS; ++q) add_vec<float, VEC>(acc, tab[v * 256 + q * L + ln]);
        float* p = a.head + ((int64_t)blockIdx.x * a.V + v) * a.D + col;
        if (on) {
#pragma unroll
            for (int c = 0; c < VEC; ++c) p[c] = acc[c];
        }
    }
    if (blockIdx.y == 0 && (uint32_t)tid < a.V) a.named[(int64_t)blockIdx.x * a.V + tid] = named[tid];
}

template <typename OT, typename I, int VEC>
__global__ __launch_bounds__(1024) void embed_table_join_kernel(const SumArgs<I> a) {
    __shared__ Vec<float, VEC> part[1024];
    const int tid = threadIdx.x, L = a.lanes, s = tid / L, ln = tid & (L - 1), NS = 1024 / L;
    const uint32_t v = blockIdx.x, share = (a.blocks + NS - 1) / NS;
    const Cols<VEC> c(a.D, L, ln, blockIdx.y);
    const int64_t col = c.col;
    const bool on = c.on;
    float acc[VEC] = {};
    int hit = 0;
    const uint32_t b1 = min(a.blocks, (s + 1) * share);
#pragma unroll 8
    for (uint32_t b = s * share; b < b1; ++b) {
        hit |= a.named[(int64_t)b * a.V + v];
        const float* p = a.head + ((int64_t)b * a.V + v) * a.D + col;
        if (on) {
#pragma unroll
            for (int c = 0; c < VEC; ++c) acc[c] += p[c];
        }
    }
    hit = __syncthreads_or(hit);
    sum_subgroups<VEC>(part, acc, L, NS);
    if (s != 0 || !on) return;
    if (hit)
        put_row<OT, VEC>(a, v, c, acc);
    else if (!a.accumulate)
        put_zeros<OT, VEC>(a, v, c);
}

// ---- the general form: every subgroup walks `run` consecutive entries of the sorted list, and a
// workgroup's 256 / lanes subgroups take consecutive pieces.  Rows are stored past the caches: 500k ids
// of rows of 32 floats take 56 us in all, 64 with cached stores.  run: 16, or 8 where 16 would leave
// compute units without a workgroup.
constexpr int kSumRun = 16;

template <typename I>
__device__ __forceinline__ uint32_t sorted_id(const SumArgs<I>& a, bool asc, uint32_t i) {
    return asc ? a.ids.get(i, a.V) : a.list[i].x;
}

template <typename GT, typename OT, typename I, int VEC>
__global__ __launch_bounds__(256) void embed_sum_kernel(const SumArgs<I> a) {
    extern __shared__ uint32_t key[];         // [1 + E + 1]: the entry before, the workgroup's, the one after
    __shared__ Vec<float, VEC> part[2][256];  // [0]: run that began before the subgroup, [1]: goes on after it
    __shared__ int state[256];                // 1: has a part[0], 2: which goes on after it, 4: has a part[1]
    const int tid = threadIdx.x, L = a.lanes, s = tid / L, ln = tid & (L - 1), NS = 256 / L;
    const uint32_t E = NS * a.run, block = xcd_remap(blockIdx.x, gridDim.x);
    uint32_t* pos = key + E + 2;
    const Cols<VEC> c(a.D, L, ln, blockIdx.y);
    const int64_t col = c.col;
    const bool on = c.on, asc = a.ascend && *a.ascend;
    constexpr uint32_t NONE = ~0u;
    const uint32_t i0 = block * E;
#pragma unroll
    for (uint32_t q = 0; q < kSumRun * 64 / 256; ++q) {  // E <= 64 * kSumRun
        const uint32_t k = q * 256 + tid, i = i0 + k;
        if (k >= E) break;
        uint2 e = make_uint2(NONE, 0);
        if (i < a.n) e = asc ? make_uint2(a.ids.get(i, a.V), i) : a.list[i];
        key[1 + k] = e.x;
        pos[k] = e.x < a.V ? e.y : 0;  // of entries without a row, row 0 of g is read and not used
    }
    if (tid == 0) key[0] = i0 ? sorted_id(a, asc, i0 - 1) : NONE;
    if (tid == 64) key[1 + E] = i0 + E < a.n ? sorted_id(a, asc, i0 + E) : NONE;
    __syncthreads();
    const GT* g = static_cast<const GT*>(a.g) + col;
    const int e0 = s * a.run;
    float acc[VEC] = {};
    bool head = key[e0] == key[1 + e0];  // the first run began before this subgroup
    int st = 0;
    for (int k0 = 0; k0 < a.run; k0 += 8) {
        Vec<GT, VEC> x[8];
        uint32_t id[9];
#pragma unroll
        for (int u = 0; u < 9; ++u) id[u] = key[1 + e0 + k0 + u];
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = load_vec<GT, VEC>(g + (int64_t)pos[e0 + k0 + u] * a.gstride);
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const uint32_t v = id[u];
            if (v >= a.V) continue;  // no row: nothing of it is summed
            add_vec<GT, VEC>(acc, x[u]);
            const bool goes_on = id[u + 1] == v;
            if (goes_on && k0 + u < a.run - 1) continue;
            if (head || goes_on) {
                Vec<float, VEC> o;
#pragma unroll
                for (int c = 0; c < VEC; ++c) o.v[c] = acc[c];
                part[head ? 0 : 1][tid] = o;
                st |= head ? (goes_on ? 3 : 1) : 4;
            } else if (on) {
                put_row<OT, VEC, true>(a, v, c, acc);
            }
            head = false;
#pragma unroll
            for (int c = 0; c < VEC; ++c) acc[c] = 0.0f;
        }
    }
    if (ln == 0) state[s] = st;
    __syncthreads();
    if (!on) return;
    auto keep = [&](float* to) {
        float* p = to + (int64_t)block * a.D + col;
#pragma unroll
        for (int c = 0; c < VEC; ++c) p[c] = acc[c];
    };
    if (st & 4) {  // a run that begins here and goes on: its owner adds the later subgroups' shares
#pragma unroll
        for (int c = 0; c < VEC; ++c) acc[c] = part[1][tid].v[c];
        bool open = true;
        for (int q = s + 1; q < NS && open; ++q) {
            add_vec<float, VEC>(acc, part[0][q * L + ln]);
            open = state[q] & 2;
        }
        if (open)
            keep(a.tail);
        else
            put_row<OT, VEC, true>(a, key[e0 + a.run], c, acc);
    }
    if (s == 0 && (st & 1)) {  // the run that an earlier workgroup began
#pragma unroll
        for (int c = 0; c < VEC; ++c) acc[c] = part[0][ln].v[c];
        for (int q = 1; q < NS && (state[q - 1] & 2); ++q) add_vec<float, VEC>(acc, part[0][q * L + ln]);
        keep(a.head);
    }
}

// First entry whose id is at least v, of ids that ascend: 64 probes at a time, by a whole wave.
template <typename I>
__device__ __forceinline__ uint32_t first_at_least(const SumArgs<I>& a, uint32_t v) {
    uint32_t lo = 0, hi = a.n;  // in [lo, hi]
    const uint32_t lane = threadIdx.x & 63;
    while (lo < hi) {
        const uint32_t step = (hi - lo + 63) / 64, at = lo + (lane + 1) * step - 1;
        const uint32_t k = __popcll(__ballot(at < hi && a.ids.get(at, a.V) < v));  // these probes come first
        hi = min(hi, lo + (k + 1) * step - 1);
        lo += k * step;
    }
    return lo;
}

// The zeros of a table whose ids came in order, by workgroups of the joining launch: `rows` rows, those
// that no id names.  (Nothing is then stored twice: a launch of the sort leaves the zeros out once it
// knows.)
template <typename OT, int VEC, typename I>
__device__ __forceinline__ void zero_between(const SumArgs<I>& a, uint32_t r0) {
    __shared__ uint8_t named[kFewRows];
    __shared__ uint32_t range[2];
    const int tid = threadIdx.x, w = tid >> 6, L = a.lanes, s = tid / L, ln = tid & (L - 1), NS = 256 / L;
    if (w < 2) {
        const uint32_t e = first_at_least(a, min(a.V, r0 + w * a.rows));
        if ((tid & 63) == 0) range[w] = e;
    }
    for (uint32_t k = tid; k < a.rows; k += 256) named[k] = 0;
    __syncthreads();
    const uint32_t e0 = range[0], e1 = range[1];
    if (e1 - e0 <= 16 * a.rows) {
        for (uint32_t e = e0 + tid; e < e1; e += 256) named[a.ids.get(e, a.V) - r0] = 1;
    } else {  // rows that are named very often: one search per row
        for (uint32_t k = tid; k < a.rows; k += 256) {
            uint32_t lo = e0, hi = e1;
            while (lo < hi) {
                const uint32_t mid = lo + ((hi - lo) >> 1);
                if (a.ids.get(mid, a.V) < r0 + k)
                    lo = mid + 1;
                else
                    hi = mid;
            }
            named[k] = lo < e1 && a.ids.get(lo, a.V) == r0 + k;
        }
    }
    __syncthreads();
    const Cols<VEC> c(a.D, L, ln, blockIdx.y);
    for (uint32_t k = s; k < a.rows && r0 + k < a.V; k += NS)
        if (c.on && !named[k]) put_zeros<OT, VEC, true>(a, r0 + k, c);
}

// The last workgroup whose first entry is v's, lo's being one (the list is sorted); by a whole wave.
template <typename I>
__device__ __forceinline__ uint32_t last_with(const SumArgs<I>& a, bool asc, uint32_t E, uint32_t v, uint32_t lo) {
    uint32_t hi = a.blocks;  // v's at lo, not at hi
    const uint32_t lane = threadIdx.x & 63;
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 63) / 64, at = lo + (lane + 1) * step;
        const uint32_t k = __popcll(__ballot(at < hi && sorted_id(a, asc, at * E) == v));  // these come first
        hi = min(hi, lo + (k + 1) * step);
        lo += k * step;
    }
    return lo;
}

// The sums of a run that begins in workgroup b and reaches into b + 1 .. b + m: b's tail and the others'
// heads, each subgroup of the 256 / lanes a consecutive share, joined through LDS.
template <typename OT, int VEC, typename I>
__device__ __forceinline__ void join_run(const SumArgs<I>& a, uint32_t v, uint32_t b, uint32_t m, int L,
                                         const Cols<VEC>& c) {
    __shared__ Vec<float, VEC> part[256];
    const int s = threadIdx.x / L, NS = 256 / L;
    const uint32_t share = (m + NS - 1) / NS;
    float acc[VEC] = {};
    if (c.on) {
        const uint32_t j0 = b + 1 + min(m, s * share), j1 = b + 1 + min(m, (s + 1) * share);
#pragma unroll 8
        for (uint32_t j = j0; j < j1; ++j) {
            const float* p = a.head + (int64_t)j * a.D + c.col;
#pragma unroll
            for (int k = 0; k < VEC; ++k) acc[k] += p[k];
        }
    }
    if (c.on && s == 0) {
        const float* p = a.tail + (int64_t)b * a.D + c.col;
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] += p[k];
    }
    sum_subgroups<VEC>(part, acc, L, m < (uint32_t)NS ? (int)m : NS);
    if (s == 0 && c.on) put_row<OT, VEC>(a, v, c, acc);
}

// One workgroup per workgroup of the sums: if a run begins in it and goes on, into at most kLong others,
// it joins the run's sums.  Longer runs cross the start of a workgroup whose number kLong divides: for each of
// those there are workgroups of strips of 8 lanes' columns, so that a long run's many heads are read by
// many units (100k rows of 256 bf16 that are all one row's: 7.9 us, 35.5 by one workgroup).
constexpr uint32_t kLong = 64;  // a wave's lanes
constexpr int kStripLanes = 8;

template <typename OT, typename I, int VEC>
__global__ __launch_bounds__(256) void embed_join_kernel(const SumArgs<I> a, uint32_t zero_blocks) {
    __shared__ uint32_t s_run[2];
    const int tid = threadIdx.x, L = a.lanes, ln = tid & (L - 1), NS = 256 / L;
    const bool asc = a.ascend && *a.ascend;
    const uint32_t E = NS * a.run;
    uint32_t b = blockIdx.x;
    if (b >= a.blocks + zero_blocks) {
        constexpr int SV = VEC < 4 ? VEC : 4;
        const uint32_t strips = (uint32_t)((a.D + kStripLanes * SV - 1) / (kStripLanes * SV));
        const uint32_t k = (b - a.blocks - zero_blocks) * gridDim.y + blockIdx.y, at = (k / strips + 1) * kLong;
        if (at >= a.blocks) return;
        const uint32_t v = sorted_id(a, asc, at * E), from = at - kLong;
        if (v >= a.V || sorted_id(a, asc, at * E - 1) != v) return;
        if (from && sorted_id(a, asc, from * E) == v && sorted_id(a, asc, from * E - 1) == v) return;  // an earlier one's
        if (tid < 64) {  // the first workgroup that ends with v
            const uint64_t ends = __ballot(sorted_id(a, asc, (from + tid + 1) * E - 1) == v);
            const uint32_t last = last_with(a, asc, E, v, at);
            if (tid == 0) {
                s_run[0] = from + __ffsll((unsigned long long)ends) - 1;
                s_run[1] = last;
            }
        }
        __syncthreads();
        b = s_run[0];
        const uint32_t m = s_run[1] - b;
        const Cols<SV> c(a.D, kStripLanes, tid & (kStripLanes - 1), k % strips);
        if (m > kLong) join_run<OT, SV>(a, v, b, m, kStripLanes, c);
        return;
    }
    if (b >= a.blocks) {
        if (asc) zero_between<OT, VEC>(a, (b - a.blocks) * a.rows);
        return;
    }
    const uint32_t i0 = b * E, i1 = i0 + E;
    if (i1 >= a.n) return;
    const uint32_t v = sorted_id(a, asc, i1), v1 = sorted_id(a, asc, i1 - 1), v0 = sorted_id(a, asc, b ? i0 - 1 : i1);
    if (v >= a.V || v1 != v || (b && v0 == v)) return;
    if (tid < 64) {
        const uint32_t last = last_with(a, asc, E, v, b + 1);
        if (tid == 0) s_run[0] = last;
    }
    __syncthreads();
    const uint32_t m = s_run[0] - b;
    if (m <= kLong) join_run<OT, VEC>(a, v, b, m, L, Cols<VEC>(a.D, L, ln, blockIdx.y));
}

// ---------------------------------------------------------------------------------- launches

enum BwdForm { kFew, kTable, kBucket, kRadix };

struct BwdPlan {
    BwdForm form;
    int lanes, run, shift, passes, bits;
    uint32_t buckets, tiles, blocks, slabs, rows;
    size_t list_a, list_b, hist, total, ascend, head, tail, named, bytes;
};

static BwdPlan bwd_plan(int64_t V, int64_t n, int64_t D, int vec) {
    BwdPlan p{};
    const int64_t per_row = (D + vec - 1) / vec;
    p.lanes = 4;  // at least: 64 subgroups per workgroup at most
    while (p.lanes < 64 && p.lanes < per_row) p.lanes <<= 1;
    const int64_t NS = 256 / p.lanes;
    p.slabs = (uint32_t)((per_row + p.lanes - 1) / p.lanes);
    size_t o = 0;
    auto take = [&](size_t b) {
        const size_t at = o;
        o += align256(b);
        return at;
    };
    const int64_t bucket_most = V >> kSortBits ? kBucketMost : kBucketMostOfOne;
    p.form = n <= kFewMost ? kFew : V * vec <= kTableMost ? kTable : n <= bucket_most ? kBucket : kRadix;
    if (p.form == kTable) {
        int64_t blocks = (V * vec > 64 ? 256 : 512) / p.slabs;  // as many as the tables leave room for
        if (blocks < 1) blocks = 1;
        const int64_t step = kTableRounds * NS, rows = (n + blocks - 1) / blocks;
        p.rows = (uint32_t)((rows + step - 1) / step * step);
        p.blocks = (uint32_t)((n + p.rows - 1) / p.rows);
        p.head = take((size_t)p.blocks * V * D * 4);
        p.named = take((size_t)p.blocks * V);
    } else if (p.form != kFew) {
        p.run = (n / (NS * kSumRun) + 1) * p.slabs < 256 ? 8 : kSumRun;
        p.blocks = (uint32_t)((n + NS * p.run - 1) / (NS * p.run));
        p.list_a = take((size_t)n * 8);
        if (n > kBucketKeep) p.list_b = take((size_t)n * 8);
        p.head = take((size_t)p.blocks * D * 4);
        p.tail = take((size_t)p.blocks * D * 4);
        int key_bits = 1;
        while ((V >> key_bits) != 0) ++key_bits;  // ids 0 .. V (V: no row)
        if (p.form == kBucket) {
            p.shift = key_bits > kBucketLog ? key_bits - kBucketLog : 0;
            p.buckets = (uint32_t)(V >> p.shift) + 1;
            key_bits = p.shift;
        }
        const int most = p.form == kBucket ? kBucketBits : kSortBits;
        p.passes = (key_bits + most - 1) / most;
        p.bits = p.passes ? (key_bits + p.passes - 1) / p.passes : 0;
        if (p.form == kRadix) {
            p.tiles = (uint32_t)((n + kSortTile - 1) / kSortTile);
            p.hist = take(((size_t)p.tiles << p.bits) * 4);
            p.total = take((4ull << p.bits));
            p.ascend = take(((size_t)p.tiles + 1) * 4);
        }
    }
    p.bytes = o;
    return p;
}

// the zeros of a dense gradient
static ZeroPart all_zeros(void* dw, size_t bytes) {
    ZeroPart z{};
    char *p = static_cast<char*>(dw), *end = p + bytes;
    size_t before = (16 - (uintptr_t)p % 16) % 16;
    if (before > bytes) before = bytes;
    z.p = reinterpret_cast<uint4*>(p + before);
    z.units = (int64_t)(bytes - before) / 16;
    z.edge[0] = reinterpret_cast<uint16_t*>(p);
    z.nedge[0] = (int)before / 2;
    z.edge[1] = reinterpret_cast<uint16_t*>(z.p + z.units);
    z.nedge[1] = (int)(end - reinterpret_cast<char*>(z.p + z.units)) / 2;
    return z;
}
// part k of `parts`, and its workgroups (none of a sum that is added to a table: z.p is null)
static ZeroPart take_zeros(const ZeroPart& z, int k, int parts, uint32_t& blocks) {
    blocks = 0;
    if (!z.p) return z;
    ZeroPart part = z;
    const int64_t u0 = z.units * k / parts, u1 = z.units * (k + 1) / parts;
    part.p = z.p + u0;
    part.units = u1 - u0;
    if (k) part.nedge[0] = part.nedge[1] = 0;
    const int64_t want = (part.units + kZeroUnits - 1) / kZeroUnits;
    blocks = (uint32_t)(want < 1 << 20 ? want : 1 << 20);  // a launch holds fewer than 2^32 threads
    if (k == 0 && blocks == 0) blocks = 1;
    return part;
}

// sorts the ids: a.list, or a.ascend where they may turn out to be sorted
template <typename I>
static void launch_sort(const BwdPlan& p, char* w, SumArgs<I>& a, const ZeroPart& z, hipStream_t s) {
    uint2 *la = reinterpret_cast<uint2*>(w + p.list_a), *lb = reinterpret_cast<uint2*>(w + p.list_b);
    uint32_t zb, zb1;
    if (p.form == kBucket) {
        const ZeroPart all = take_zeros(z, 0, 1, zb);
        const BucketArgs<I> t{a.n, a.V, a.ids, p.shift, p.passes, p.bits, p.buckets, la, lb};
        hipLaunchKernelGGL((sort_bucket_kernel<I>), dim3(p.buckets + zb), dim3(1024), 0, s, t, all);
        a.list = la;
        return;
    }
    SortArgs<I> t{};
    t.n = a.n;
    t.V = a.V;
    t.ids = a.ids;
    t.bits = p.bits;
    t.tiles = p.tiles;
    t.hist = reinterpret_cast<uint32_t*>(w + p.hist);
    t.total = reinterpret_cast<uint32_t*>(w + p.total);
    t.ascend = reinterpret_cast<uint32_t*>(w + p.ascend);
    const unsigned scan_blocks = ((1u << p.bits) + 63) / 64;
    const int parts = 2 * p.passes - 1;
    for (int pass = 0; pass < p.passes; ++pass) {
        t.in = pass == 0 ? nullptr : pass & 1 ? la : lb;
        t.out = pass & 1 ? lb : la;
        t.shift = pass * p.bits;
        // zeros from the first scatter on, where it is known whether the ids ascend
        ZeroPart z0{};
        if (pass) z0 = take_zeros(z, 2 * pass - 1, parts, zb);
        const ZeroPart z1 = take_zeros(z, 2 * pass, parts, zb1);
        if (pass == 0) {
            hipLaunchKernelGGL((sort_count_kernel<true, I>), dim3(p.tiles), dim3(256), 0, s, t, z0);
            hipLaunchKernelGGL((sort_scan_kernel<true, I>), dim3(scan_blocks + 1), dim3(1024), 0, s, t);
            hipLaunchKernelGGL((sort_scatter_kernel<true, I>), dim3(p.tiles + zb1), dim3(256), 0, s, t, z1);
        } else {
            hipLaunchKernelGGL((sort_count_kernel<false, I>), dim3(p.tiles + zb), dim3(256), 0, s, t, z0);
            hipLaunchKernelGGL((sort_scan_kernel<false, I>), dim3(scan_blocks), dim3(1024), 0, s, t);
            hipLaunchKernelGGL((sort_scatter_kernel<false, I>), dim3(p.tiles + zb1), dim3(256), 0, s, t, z1);
        }
    }
    a.list = t.out;
    a.ascend = t.ascend;
}

template <typename GT, typename OT, int VEC, typename I>
static void launch_sums(const BwdPlan& p, const SumArgs<I>& a, uint32_t zero_blocks, hipStream_t s) {
    const dim3 block(256);
    switch (p.form) {
        case kFew:
            hipLaunchKernelGGL((embed_few_kernel<GT, OT, I, VEC>), dim3(a.n + zero_blocks, p.slabs), block, 0, s, a);
            break;
        case kTable:
            hipLaunchKernelGGL((embed_table_kernel<GT, I, VEC>), dim3(a.blocks, p.slabs), block,
                               (size_t)a.V * 256 * VEC * sizeof(float), s, a);
            hipLaunchKernelGGL((embed_table_join_kernel<OT, I, VEC>), dim3(a.V, p.slabs), dim3(1024), 0, s,
                               a);
            break;
        default:
            hipLaunchKernelGGL((embed_sum_kernel<GT, OT, I, VEC>), dim3(a.blocks, p.slabs), block,
                               (2 * (256 / a.lanes) * a.run + 2) * sizeof(uint32_t), s, a);
            if (a.blocks + zero_blocks > 1) {
                constexpr int strip = kStripLanes * (VEC < 4 ? VEC : 4);
                const uint64_t strips = (uint64_t)((a.D + strip - 1) / strip) * ((a.blocks - 1) / kLong);
                const uint32_t longs = (uint32_t)((strips + p.slabs - 1) / p.slabs);
                hipLaunchKernelGGL((embed_join_kernel<OT, I, VEC>), dim3(a.blocks + zero_blocks + longs, p.slabs), block, 0,
                                   s, a, zero_blocks);
            }
    }
}

template <typename GT, typename OT, typename I>
static void launch_sums(int vec, const BwdPlan& p, const SumArgs<I>& a, uint32_t zero_blocks, hipStream_t s) {
    switch (vec) {
        case 8: return launch_sums<GT, OT, sizeof(GT) == 4 ? 4 : 8>(p, a, zero_blocks, s);
        case 4: return launch_sums<GT, OT, 4>(p, a, zero_blocks, s);
        case 2: return launch_sums<GT, OT, 2>(p, a, zero_blocks, s);
        default: return launch_sums<GT, OT, 1>(p, a, zero_blocks, s);
    }
}

template <typename GT, typename I>
static void launch_sums(int dwtype, int vec, const BwdPlan& p, const SumArgs<I>& a, uint32_t zero_blocks,
                        hipStream_t s) {
    if (dwtype == HGSR_F32) return launch_sums<GT, float>(vec, p, a, zero_blocks, s);
    if (dwtype == HGSR_F16) return launch_sums<GT, f16_t>(vec, p, a, zero_blocks, s);
    return launch_sums<GT, bf16_t>(vec, p, a, zero_blocks, s);
}

template <typename I>
static int launch_bwd(const BwdPlan& p, char* w, SumArgs<I> a, const void* ids, int64_t ids_stride, int gtype,
                      int dwtype, int vec, hipStream_t s) {
    a.ids = RowIds<I>{static_cast<const I*>(ids), ids_stride};
    KernelTimer kt("embed_bwd", s);
    uint32_t zero_blocks = 0;
    const size_t dw_bytes = (size_t)a.V * a.D * elem_size(dwtype);
    if ((p.form == kFew || p.form == kRadix) && !a.accumulate) {  // about 32 KB of zeros per workgroup
        int64_t rows = 32768 / ((int64_t)p.lanes * vec * elem_size(dwtype));
        while (a.V / rows > 1 << 23) rows *= 2;  // a launch holds fewer than 2^24 workgroups
        a.rows = (uint32_t)(rows > kFewRows ? kFewRows : rows);
        zero_blocks = (a.V + a.rows - 1) / a.rows;
    }
    if (p.form == kBucket || p.form == kRadix)
        launch_sort(p, w, a, a.accumulate ? ZeroPart{} : all_zeros(a.dw, dw_bytes), s);
    if (gtype == HGSR_F32)
        launch_sums<float>(dwtype, vec, p, a, zero_blocks, s);
    else if (gtype == HGSR_F16)
        launch_sums<f16_t>(dwtype, vec, p, a, zero_blocks, s);
    else
        launch_sums<bf16_t>(dwtype, vec, p, a, zero_blocks, s);
    return check_launch("embed_bwd");
}

struct FwdArgs {
    int64_t V, n, D, wstride, ids_stride;
    const void *w, *ids;
    int ids64;
    float scale;
    void* out;
};

template <typename WT, typename OT, typename I, int VEC, bool STREAM>
static void launch_fwd(const FwdArgs& a, hipStream_t s) {
    const uint32_t per_row = (uint32_t)((a.D + VEC - 1) / VEC);
    const RowIds<I> ids{static_cast<const I*>(a.ids), a.ids_stride};
    const int64_t most = ((int64_t)1 << 30) / per_row;  // rows per launch: at most 2^30 pieces
    for (int64_t r0 = 0; r0 < a.n; r0 += most) {
        const uint32_t chunks = (uint32_t)((a.n - r0 < most ? a.n - r0 : most) * per_row);
        hipLaunchKernelGGL((embed_fwd_kernel<WT, OT, I, VEC, STREAM>), dim3((chunks + 255) / 256), dim3(256), 0, s, chunks,
                           fast_div(per_row), (uint32_t)a.V, (uint32_t)a.D, static_cast<const WT*>(a.w),
                           a.wstride, ids, r0, a.scale, static_cast<OT*>(a.out));
    }
}

template <typename WT, typename OT, typename I, int VEC>
static void launch_fwd(const FwdArgs& a, hipStream_t s) {
    return stream_out(a.n * a.D * (int64_t)sizeof(OT)) ? launch_fwd<WT, OT, I, VEC, true>(a, s)
                                                       : launch_fwd<WT, OT, I, VEC, false>(a, s);
}

template <typename WT, typename OT, typename I>
static void launch_fwd(int vec, const FwdArgs& a, hipStream_t s) {
    switch (vec) {
        case 8: return launch_fwd<WT, OT, I, sizeof(WT) + sizeof(OT) == 4 ? 8 : 4>(a, s);
        case 4: return launch_fwd<WT, OT, I, 4>(a, s);
        case 2: return launch_fwd<WT, OT, I, 2>(a, s);
        default: return launch_fwd<WT, OT, I, 1>(a, s);
    }
}

template <typename WT, typename OT>
static void launch_fwd(int vec, const FwdArgs& a, hipStream_t s) {
    return a.ids64 ? launch_fwd<WT, OT, int64_t>(vec, a, s) : launch_fwd<WT, OT, int32_t>(vec, a, s);
}

template <typename WT>
static void launch_fwd(int otype, int vec, const FwdArgs& a, hipStream_t s) {
    if (otype == HGSR_F32) return launch_fwd<WT, float>(vec, a, s);
    if (otype == HGSR_F16) return launch_fwd<WT, f16_t>(vec, a, s);
    return launch_fwd<WT, bf16_t>(vec, a, s);
}

}  // namespace hgsr

using namespace hgsr;

static int check_dims(const char* what, int64_t V, int64_t n, int64_t D) {
    HGSR_REQUIRE(V >= 0 && V < (1ll << 31), "%s: rows %lld outside [0, 2^31)", what, (long long)V);
    HGSR_REQUIRE(n >= 0 && n < (1ll << 31) - 4096, "%s: %lld ids: at most 2^31 - 4097", what, (long long)n);
    HGSR_REQUIRE(D >= 1 && D <= (1ll << 21), "%s: row length %lld outside [1, 2^21]", what, (long long)D);
    return HGSR_OK;
}

extern "C" int hgsr_embed_fwd(int64_t V, int64_t n, int64_t D, const void* weight, int wtype, int64_t wstride,
                              const void* ids, int ids64, int64_t ids_stride, float scale, void* out, int otype,
                              hgsr_stream_t stream) {
    if (int st = check_dims("embed_fwd", V, n, D)) return st;
    HGSR_REQUIRE(type_ok(wtype) && type_ok(otype), "embed_fwd: unknown element type");
    HGSR_REQUIRE(wstride >= 0 && ids_stride >= 0, "embed_fwd: negative stride");
    if (n == 0) return HGSR_OK;
    HGSR_REQUIRE(ids && out && (weight || V == 0), "embed_fwd: null pointer");
    const int most = wtype != HGSR_F32 && otype != HGSR_F32 ? 8 : 4;
    const int vec = vec_width(most, D);
    const FwdArgs a{V, n, D, wstride, ids_stride, weight, ids, ids64, scale, out};
    hipStream_t s = as_stream(stream);
    {
        KernelTimer kt("embed_fwd", s);
        if (wtype == HGSR_F32)
            launch_fwd<float>(otype, vec, a, s);
        else if (wtype == HGSR_F16)
            launch_fwd<f16_t>(otype, vec, a, s);
        else
            launch_fwd<bf16_t>(otype, vec, a, s);
    }
    return check_launch("embed_fwd");
}

extern "C" size_t hgsr_embed_bwd_ws_bytes(int64_t V, int64_t n, int64_t D) {
    if (V <= 0 || n <= 0 || D < 1) return 0;
    size_t most = 0;
    for (int widest = 4; widest <= 8; widest <<= 1) {  // of a 32-bit and of a 16-bit gradient
        const size_t b = bwd_plan(V, n, D, vec_width(widest, D)).bytes;
        if (b > most) most = b;
    }
    return most;
}

extern "C" int hgsr_embed_bwd(int64_t V, int64_t n, int64_t D, const void* g, int gtype, int64_t gstride,
                              const void* ids, int ids64, int64_t ids_stride, float scale, void* dw, int dwtype,
                              int64_t dwstride, int accumulate, void* ws, size_t ws_bytes, hgsr_stream_t stream) {
    if (int st = check_dims("embed_bwd", V, n, D)) return st;
    HGSR_REQUIRE(type_ok(gtype) && type_ok(dwtype), "embed_bwd: unknown element type");
    HGSR_REQUIRE(gstride >= 0 && dwstride >= D && ids_stride >= 0, "embed_bwd: bad stride");
    HGSR_REQUIRE(accumulate || dwstride == D, "embed_bwd: bad stride: a dense gradient is contiguous");
    if (V == 0) return HGSR_OK;
    HGSR_REQUIRE(dw, "embed_bwd: null pointer");
    hipStream_t s = as_stream(stream);
    const size_t dw_bytes = (size_t)V * D * elem_size(dwtype);
    HGSR_REQUIRE(accumulate || dw_bytes >> 38 == 0, "embed_bwd: a dense gradient of %zu bytes: less than 2^38", dw_bytes);
    if (n == 0) {
        if (!accumulate) {
            uint32_t zb;
            const ZeroPart z = take_zeros(all_zeros(dw, dw_bytes), 0, 1, zb);
            hipLaunchKernelGGL(zero_kernel, dim3(zb), dim3(256), 0, s, z);
        }
        return check_launch("embed_bwd");
    }
    HGSR_REQUIRE(g && ids, "embed_bwd: null pointer");
    const int most = gtype == HGSR_F32 ? 4 : 8;
    const int vec = vec_width(most, D);
    const BwdPlan p = bwd_plan(V, n, D, vec);
    if (p.bytes > ws_bytes || (p.bytes && !ws)) {
        set_error("embed_bwd: workspace of %zu bytes, %zu needed", ws ? ws_bytes : (size_t)0, p.bytes);
        return HGSR_EWORKSPACE;
    }
    HGSR_REQUIRE(p.blocks <= (1u << 22), "embed_bwd: %lld ids of rows of %lld: too many for a launch", (long long)n,
                 (long long)D);
    char* w = static_cast<char*>(ws);
    auto run = [&](auto none) {
        SumArgs<decltype(none)> a{};
        a.n = (uint32_t)n;
        a.V = (uint32_t)V;
        a.D = D;
        a.g = g;
        a.gstride = gstride;
        a.dw = dw;
        a.dwstride = dwstride;
        a.accumulate = accumulate != 0;
        a.scale = scale;
        a.lanes = p.lanes;
        a.run = p.run;
        a.blocks = p.blocks;
        a.rows = p.rows;
        a.head = reinterpret_cast<float*>(w + p.head);
        a.tail = reinterpret_cast<float*>(w + p.tail);
        a.named = reinterpret_cast<uint8_t*>(w + p.named);
        return launch_bwd(p, w, a, ids, ids_stride, gtype, dwtype, vec, s);
    };
    return ids64 ? run(int64_t{}) : run(int32_t{});
}
