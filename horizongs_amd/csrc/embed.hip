// K18: embedding lookup with scaling, and its gradient by sorted ids (the per-camera appearance
// rows of the reference, scene/embedding.py:50-79, and any other table of learned rows).
//
//   out[i, :] = scale * W[ids[i], :]                       (zeros where ids[i] is no row of W)
//   dW[v, :]  = scale * sum over i with ids[i] = v of g[i, :]
//
// The lookup is a gather: one 16-byte piece of a row per lane.
//
// The gradient is summed in a fixed order, without float atomics, so it is the same bits on every
// run: the (id, i) pairs are sorted by id (stable), the sorted list is cut into equal pieces -- not
// into rows, so a row named by half of the entries costs no more than any other -- and each piece
// sums its runs in f32.  Runs inside a piece are written at once; the pieces' first and last runs
// are joined through LDS inside a workgroup and through a workspace between workgroups.
#include "rows.h"

namespace hgsr {

// ------------------------------------------------------------------------------------- lookup

constexpr int kFwdPer = 4;  // pieces per lane, 256 apart

template <typename WT, typename OT, int VEC>
__global__ __launch_bounds__(256) void embed_fwd_kernel(uint32_t chunks, FastDiv per_row, uint32_t V,
                                                        const WT* __restrict__ w, int64_t wstride, RowIds ids,
                                                        int64_t row0, float scale, OT* __restrict__ out) {
    const uint32_t c0 = xcd_remap(blockIdx.x, gridDim.x) * (256 * kFwdPer) + threadIdx.x;
    uint32_t col[kFwdPer], id[kFwdPer], row[kFwdPer];
#pragma unroll
    for (int k = 0; k < kFwdPer; ++k) {
        const uint32_t c = c0 + k * 256;
        row[k] = per_row.div(c < chunks ? c : 0);
        col[k] = (c - row[k] * per_row.d) * VEC;
        id[k] = ids.get(row0 + row[k], V);
    }
    Vec<WT, VEC> x[kFwdPer];
#pragma unroll
    for (int k = 0; k < kFwdPer; ++k)
        if (c0 + k * 256 < chunks && id[k] < V) x[k] = load_vec<WT, VEC>(w + (int64_t)id[k] * wstride + col[k]);
#pragma unroll
    for (int k = 0; k < kFwdPer; ++k) {
        if (c0 + k * 256 >= chunks) break;
        Vec<OT, VEC> o;
#pragma unroll
        for (int j = 0; j < VEC; ++j) o.v[j] = (OT)(id[k] < V ? (float)x[k].v[j] * scale : 0.0f);
        store_vec<OT, VEC>(out + (row0 + row[k]) * ((int64_t)per_row.d * VEC) + col[k], o);
    }
}

// --------------------------------------------------------------------------- zeros of the table
// A dense gradient's zeros are stored by extra workgroups of the launches that sort the ids: the
// sort is a chain of short, latency-bound kernels, and the memory is free meanwhile.  Rows that an
// id names are stored again by the sums.
struct ZeroPart {
    uint4* p;        // whole 16-byte units
    int64_t units;
    uint16_t* edge[2];  // what lies before the first and behind the last unit (part 0 only)
    int nedge[2];
};
constexpr int kZeroUnits = 2048;  // per workgroup: 32 KB

__device__ __forceinline__ void store_zeros(const ZeroPart& z, int64_t block) {
    const int64_t u0 = block * kZeroUnits + threadIdx.x;
#pragma unroll
    for (int k = 0; k < kZeroUnits / 256; ++k)
        if (u0 + k * 256 < z.units) z.p[u0 + k * 256] = make_uint4(0, 0, 0, 0);
    if (block == 0 && threadIdx.x < 8) {
        if ((int)threadIdx.x < z.nedge[0]) z.edge[0][threadIdx.x] = 0;
        if ((int)threadIdx.x < z.nedge[1]) z.edge[1][threadIdx.x] = 0;
    }
}

__global__ __launch_bounds__(256) void zero_kernel(ZeroPart z) { store_zeros(z, blockIdx.x); }

// ------------------------------------------------------------------------------ sort of (id, i)
// Up to kRankMost entries: the place of each is the number of entries before it, counted by
// comparing it with all of them -- n^2 comparisons over the whole chip, in one launch.
constexpr int kRankMost = 16384;
constexpr int kRankOwn = 4;      // entries per wave
constexpr int kRankTile = 2048;  // ids staged in LDS at a time

__global__ __launch_bounds__(256) void sort_rank_kernel(uint32_t n, RowIds ids, uint32_t V, uint2* __restrict__ out,
                                                        uint32_t blocks, ZeroPart zeros) {
    __shared__ uint32_t key[kRankTile];
    if (blockIdx.x >= blocks) return store_zeros(zeros, blockIdx.x - blocks);
    const int lane = threadIdx.x & 63;
    const uint32_t i0 = __builtin_amdgcn_readfirstlane((blockIdx.x * 4 + (threadIdx.x >> 6)) * kRankOwn);
    uint32_t mine[kRankOwn], before[kRankOwn] = {};
#pragma unroll
    for (int q = 0; q < kRankOwn; ++q)
        mine[q] = __builtin_amdgcn_readfirstlane(i0 + q < n ? ids.get(i0 + q, V) : 0);
    for (uint32_t j0 = 0; j0 < n; j0 += kRankTile) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kRankTile / 256; ++k) {
            const uint32_t j = j0 + k * 256 + threadIdx.x;
            key[k * 256 + threadIdx.x] = j < n ? ids.get(j, V) : ~0u;
        }
        __syncthreads();
        if (j0 + kRankTile <= i0 || j0 >= i0 + kRankOwn) {  // all before or all behind this wave's entries
            const uint32_t tie = j0 < i0 ? 1 : 0;           // an equal id counts if it comes before
#pragma unroll 8
            for (int k = 0; k < kRankTile; k += 64) {
                const uint32_t v = key[k + lane];
#pragma unroll
                for (int q = 0; q < kRankOwn; ++q) before[q] += v < mine[q] + tie;
            }
        } else {
            for (int k = 0; k < kRankTile; k += 64) {
                const uint32_t v = key[k + lane], j = j0 + k + lane;
#pragma unroll
                for (int q = 0; q < kRankOwn; ++q) before[q] += v < mine[q] || (v == mine[q] && j < i0 + q);
            }
        }
    }
#pragma unroll
    for (int q = 0; q < kRankOwn; ++q) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) before[q] += __shfl_xor(before[q], d);
        if (lane == q && i0 + q < n) out[before[q]] = make_uint2(mine[q], i0 + q);
    }
}

// More: least-significant-digit radix sort, digits of up to 11 bits.  Per pass: the tiles' digit
// counts, their prefix over the tiles, a stable scatter.  The first pass also notes whether the
// ids ascend already (a compacted index does): the rest of the sort then ends at once, and the
// sums read the ids themselves.
constexpr int kSortRounds = 8;
constexpr int kSortTile = 256 * kSortRounds;  // entries per workgroup: 4 waves x 8 rounds x 64 lanes
constexpr int kSortBits = 11;

struct SortArgs {
    uint32_t n, V;
    RowIds ids;
    const uint2* in;   // nullptr: the first pass, entries from the ids
    uint2* out;
    int shift, bits;
    uint32_t tiles;
    uint32_t* hist;    // [tiles][1 << bits]
    uint32_t* total;   // [1 << bits]
    uint32_t* ascend;  // [1 + tiles]: the verdict, then the tiles' own
};

template <bool FIRST>
__device__ __forceinline__ uint2 sort_entry(const SortArgs& a, uint32_t i) {
    if (FIRST) return make_uint2(a.ids.get(i, a.V), i);
    return a.in[i];
}

template <bool FIRST>
__global__ __launch_bounds__(256) void sort_count_kernel(const SortArgs a, ZeroPart zeros) {
    __shared__ uint32_t h[1 << kSortBits];
    if (blockIdx.x >= a.tiles) return store_zeros(zeros, blockIdx.x - a.tiles);
    if (!FIRST && *a.ascend) return;
    const uint32_t bins = 1u << a.bits, base = blockIdx.x * kSortTile;
    uint32_t v[kSortRounds], next[kSortRounds];
#pragma unroll
    for (int k = 0; k < kSortRounds; ++k) {
        const uint32_t i = base + k * 256 + threadIdx.x;
        if (i < a.n) v[k] = sort_entry<FIRST>(a, i).x;
        if (FIRST) next[k] = i + 1 < a.n ? a.ids.get(i + 1, a.V) : ~0u;
    }
    for (uint32_t b = threadIdx.x; b < bins; b += 256) h[b] = 0;
    __syncthreads();
    int up = 1;
#pragma unroll
    for (int k = 0; k < kSortRounds; ++k)
        if (base + k * 256 + threadIdx.x < a.n) {
            atomicAdd(&h[(v[k] >> a.shift) & (bins - 1)], 1u);
            if (FIRST) up &= v[k] <= next[k];
        }
    up = __syncthreads_and(up);
    if (FIRST && threadIdx.x == 0) a.ascend[1 + blockIdx.x] = up;
    for (uint32_t b = threadIdx.x; b < bins; b += 256) a.hist[(size_t)blockIdx.x * bins + b] = h[b];
}

// 64 digits per workgroup, a share of the tiles per wave: exclusive prefix of each digit's counts
// over the tiles, and its total.  The last workgroup of the first pass joins the tiles' verdicts.
template <bool FIRST>
__global__ __launch_bounds__(1024) void sort_scan_kernel(const SortArgs a) {
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

template <bool FIRST>
__global__ __launch_bounds__(256) void sort_scatter_kernel(const SortArgs a, ZeroPart zeros) {
    __shared__ uint32_t cnt[4][1 << kSortBits];  // per wave: count, then where its entries of the digit go
    __shared__ uint32_t wsum[4];
    if (blockIdx.x >= a.tiles) return store_zeros(zeros, blockIdx.x - a.tiles);
    if (*a.ascend) return;
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
    // the lanes of this wave whose digit equals mine; the first of them adds their number
    uint64_t same[kSortRounds];
    uint32_t old[kSortRounds];
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
        const bool on = base + r * 64 + lane < a.n;
        const uint32_t d = (e[r].x >> a.shift) & (bins - 1);
        uint64_t s = __ballot(on);
        if (!on) s = ~s;
#pragma unroll
        for (int k = 0; k < kSortBits; ++k)
            if (k < a.bits) {
                const uint64_t m = __ballot((d >> k) & 1);
                s &= (d >> k) & 1 ? m : ~m;
            }
        same[r] = s;
        old[r] = 0;
        if (on && (s & ((1ull << lane) - 1)) == 0) old[r] = atomicAdd(&cnt[w][d], (uint32_t)__popcll(s));
    }
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r)  // the entry's place among the wave's entries of its digit
        old[r] = __shfl(old[r], __ffsll((unsigned long long)same[r]) - 1) + __popcll(same[r] & ((1ull << lane) - 1));
    uint32_t inc = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(inc, d);
        if (lane >= d) inc += o;
    }
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
struct SumArgs {
    uint32_t n, V;
    int64_t D;
    RowIds ids;
    const uint2* list;       // sorted (id, i)
    const uint32_t* ascend;  // not null and set: the ids ascend by themselves, no list was made
    const void* g;
    int64_t gstride;
    void* dw;
    int64_t dwstride;
    int dwtype, accumulate;
    float scale;
    int lanes;           // lanes per subgroup, a power of two
    uint32_t blocks;     // workgroups over the entries
    float *head, *tail;  // [blocks][D]: the sums of a workgroup's runs that began before it / go on after it
    uint32_t rows;       // table form: entries per workgroup; few entries: rows per zeroing workgroup
    uint8_t* named;      // table form: [blocks][V]
};

template <int VEC>
__device__ __forceinline__ void put_row(const SumArgs& a, uint32_t v, int64_t col, const float* acc) {
    const int64_t at = (int64_t)v * a.dwstride + col;
    auto put = [&](auto* p) {
        using OT = typename std::remove_pointer<decltype(p)>::type;
        Vec<OT, VEC> o;
        if (a.accumulate) {
            o = load_vec<OT, VEC>(p);
#pragma unroll
            for (int k = 0; k < VEC; ++k) o.v[k] = (OT)((float)o.v[k] + acc[k] * a.scale);
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k) o.v[k] = (OT)(acc[k] * a.scale);
        }
        store_vec<OT, VEC>(p, o);
    };
    if (a.dwtype == HGSR_F32)
        put(static_cast<float*>(a.dw) + at);
    else if (a.dwtype == HGSR_F16)
        put(static_cast<f16_t*>(a.dw) + at);
    else
        put(static_cast<bf16_t*>(a.dw) + at);
}

template <typename T, int VEC>
__device__ __forceinline__ void add_vec(float* acc, const Vec<T, VEC>& x) {
#pragma unroll
    for (int c = 0; c < VEC; ++c) acc[c] += (float)x.v[c];
}

// ---- few entries: one launch, a workgroup per entry.  The first of the entries that name a row
// sums them all (each subgroup every NS-th of them, joined through LDS); other workgroups store the
// zeros of the rows that no id names.
constexpr int kFewMost = 256;
constexpr int kFewRows = 1024;  // rows per zeroing workgroup, at most

template <typename GT, int VEC>
__global__ __launch_bounds__(256) void embed_few_kernel(const SumArgs a) {
    __shared__ Vec<float, VEC> part[256];
    __shared__ uint32_t match[kFewMost];
    __shared__ uint32_t count[4], first[4];
    __shared__ uint8_t named[kFewRows];
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
    const int L = a.lanes, s = tid / L, ln = tid & (L - 1), NS = 256 / L;
    const int64_t col = ((int64_t)blockIdx.y * L + ln) * VEC;
    const bool on = col < a.D;
    const uint32_t mine = (uint32_t)tid < a.n ? a.ids.get(tid, a.V) : a.V;
    if (blockIdx.x >= a.n) {
        const uint32_t r0 = (blockIdx.x - a.n) * a.rows;
        for (uint32_t k = tid; k < a.rows; k += 256) named[k] = 0;
        __syncthreads();
        if (mine < a.V && mine >= r0 && mine - r0 < a.rows) named[mine - r0] = 1;
        __syncthreads();
        const float z[VEC] = {};
        for (uint32_t k = s; k < a.rows && r0 + k < a.V; k += NS)
            if (on && !named[k]) put_row<VEC>(a, r0 + k, col, z);
        return;
    }
    const uint32_t v = a.ids.get(blockIdx.x, a.V);
    if (v >= a.V) return;
    const uint64_t same = __ballot(mine == v);
    if (lane == 0) {
        count[w] = __popcll(same);
        first[w] = same ? w * 64 + __ffsll((unsigned long long)same) - 1 : ~0u;
    }
    __syncthreads();
    if (min(min(first[0], first[1]), min(first[2], first[3])) < blockIdx.x) return;
    uint32_t at = 0, m = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        if (q < w) at += count[q];
        m += count[q];
    }
    if (mine == v) match[at + __popcll(same & ((1ull << lane) - 1))] = tid;
    __syncthreads();
    float acc[VEC] = {};
    if (on) {
        const GT* g = static_cast<const GT*>(a.g) + col;
        for (uint32_t j = s; j < m; j += 8 * NS) {
            Vec<GT, VEC> x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (j + u * NS < m) x[u] = load_vec<GT, VEC>(g + (int64_t)match[j + u * NS] * a.gstride);
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (j + u * NS < m) add_vec<GT, VEC>(acc, x[u]);
        }
    }
    Vec<float, VEC> o;
#pragma unroll
    for (int c = 0; c < VEC; ++c) o.v[c] = acc[c];
    part[tid] = o;
    __syncthreads();
    if (s || !on) return;
    for (uint32_t q = 1; q < (uint32_t)NS && q < m; ++q) add_vec<float, VEC>(acc, part[q * L + ln]);
    put_row<VEC>(a, v, col, acc);
}

// ---- few rows: no sort.  Every subgroup keeps a table of sums in LDS, its own, so a workgroup's
// entries are read once and in order; the subgroups' and then the workgroups' tables are added.
constexpr int kTableMost = 64;  // V * VEC: 64 KB of LDS, two workgroups per compute unit

template <typename GT, int VEC>
__global__ __launch_bounds__(256) void embed_table_kernel(const SumArgs a) {
    extern __shared__ __align__(16) char smem[];
    Vec<float, VEC>* tab = reinterpret_cast<Vec<float, VEC>*>(smem);  // [V][256]
    __shared__ uint8_t named[kTableMost];
    const int tid = threadIdx.x, L = a.lanes, s = tid / L, ln = tid & (L - 1), NS = 256 / L;
    const int64_t col = ((int64_t)blockIdx.y * L + ln) * VEC;
    const bool on = col < a.D;
    Vec<float, VEC> zero;
#pragma unroll
    for (int c = 0; c < VEC; ++c) zero.v[c] = 0.0f;
    for (uint32_t v = 0; v < a.V; ++v) tab[v * 256 + tid] = zero;
    if (tid < kTableMost) named[tid] = 0;
    __syncthreads();
    const GT* g = static_cast<const GT*>(a.g) + col;
    const uint64_t i1 = min((uint64_t)a.n, ((uint64_t)blockIdx.x + 1) * a.rows);
    for (uint64_t i0 = (uint64_t)blockIdx.x * a.rows + s; i0 < i1; i0 += 8 * NS) {
        uint32_t id[8];
        Vec<GT, VEC> x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int64_t i = i0 + u * NS;
            id[u] = i < (int64_t)i1 ? a.ids.get(i, a.V) : a.V;
            if (on && i < (int64_t)i1) x[u] = load_vec<GT, VEC>(g + i * a.gstride);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u)
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

template <int VEC>
__global__ __launch_bounds__(256) void embed_table_join_kernel(const SumArgs a) {
    __shared__ Vec<float, VEC> part[256];
    const int tid = threadIdx.x, L = a.lanes, s = tid / L, ln = tid & (L - 1), NS = 256 / L;
    const uint32_t v = blockIdx.x, share = (a.blocks + NS - 1) / NS;
    const int64_t col = ((int64_t)blockIdx.y * L + ln) * VEC;
    const bool on = col < a.D;
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
    Vec<float, VEC> o;
#pragma unroll
    for (int c = 0; c < VEC; ++c) o.v[c] = acc[c];
    part[tid] = o;
    hit = __syncthreads_or(hit);
    if (s || !on || (a.accumulate && !hit)) return;
    for (int q = 1; q < NS && (uint32_t)q * share < a.blocks; ++q) add_vec<float, VEC>(acc, part[q * L + ln]);
    put_row<VEC>(a, v, col, acc);
}

// ---- the general form: every subgroup walks kSumRun consecutive entries of the sorted list, and a
// workgroup's 256 / lanes subgroups take consecutive pieces.
constexpr int kSumRun = 16;

__device__ __forceinline__ uint32_t sorted_id(const SumArgs& a, bool asc, uint32_t i) {
    return asc ? a.ids.get(i, a.V) : a.list[i].x;
}

template <typename GT, int VEC>
__global__ __launch_bounds__(256) void embed_sum_kernel(const SumArgs a) {
    extern __shared__ uint32_t key[];         // [1 + E + 1]: the entry before, the workgroup's, the one after
    __shared__ Vec<float, VEC> part[2][256];  // [0]: run that began before the subgroup, [1]: goes on after it
    __shared__ int state[256];                // 1: has a part[0], 2: which goes on after it, 4: has a part[1]
    const int tid = threadIdx.x, L = a.lanes, s = tid / L, ln = tid & (L - 1), NS = 256 / L;
    const uint32_t E = NS * kSumRun, block = xcd_remap(blockIdx.x, gridDim.x);
    uint32_t* pos = key + E + 2;
    const int64_t col = ((int64_t)blockIdx.y * L + ln) * VEC;
    const bool on = col < a.D, asc = a.ascend && *a.ascend;
    constexpr uint32_t NONE = ~0u;
    const uint32_t i0 = block * E;
    for (uint32_t k = tid; k < E; k += 256) {
        const uint32_t i = i0 + k;
        uint2 e = make_uint2(NONE, 0);
        if (i < a.n) e = asc ? make_uint2(a.ids.get(i, a.V), i) : a.list[i];
        key[1 + k] = e.x;
        pos[k] = e.y;
    }
    if (tid == 0) key[0] = i0 ? sorted_id(a, asc, i0 - 1) : NONE;
    if (tid == 64) key[1 + E] = i0 + E < a.n ? sorted_id(a, asc, i0 + E) : NONE;
    __syncthreads();
    const GT* g = static_cast<const GT*>(a.g) + col;
    const int e0 = s * kSumRun;
    float acc[VEC] = {};
    bool head = key[e0] == key[1 + e0];  // the first run began before this subgroup
    int st = 0;
    for (int k0 = 0; k0 < kSumRun; k0 += 8) {
        Vec<GT, VEC> x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (on && key[1 + e0 + k0 + u] < a.V) x[u] = load_vec<GT, VEC>(g + (int64_t)pos[e0 + k0 + u] * a.gstride);
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int k = e0 + k0 + u;
            const uint32_t v = key[1 + k];
            if (v >= a.V) continue;  // no row: nothing of it is summed
            add_vec<GT, VEC>(acc, x[u]);
            const bool goes_on = key[2 + k] == v;
            if (goes_on && k0 + u < kSumRun - 1) continue;
            if (head || goes_on) {
                Vec<float, VEC> o;
#pragma unroll
                for (int c = 0; c < VEC; ++c) o.v[c] = acc[c];
                part[head ? 0 : 1][tid] = o;
                st |= head ? (goes_on ? 3 : 1) : 4;
            } else if (on) {
                put_row<VEC>(a, v, col, acc);
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
            put_row<VEC>(a, key[e0 + kSumRun], col, acc);
    }
    if (s == 0 && (st & 1)) {  // the run that an earlier workgroup began
#pragma unroll
        for (int c = 0; c < VEC; ++c) acc[c] = part[0][ln].v[c];
        for (int q = 1; q < NS && (state[q - 1] & 2); ++q) add_vec<float, VEC>(acc, part[0][q * L + ln]);
        keep(a.head);
    }
}

// One workgroup per workgroup of the sums: if a run begins in it and goes on, its tail and the
// heads of the workgroups it reaches into, each subgroup a consecutive share, joined through LDS.
template <int VEC>
__global__ __launch_bounds__(256) void embed_join_kernel(const SumArgs a) {
    __shared__ Vec<float, VEC> part[256];
    __shared__ uint32_t s_last;
    const int tid = threadIdx.x, L = a.lanes, s = tid / L, ln = tid & (L - 1), NS = 256 / L;
    const bool asc = a.ascend && *a.ascend;
    const uint32_t E = NS * kSumRun, b = blockIdx.x, i0 = b * E, i1 = i0 + E;
    if (i1 >= a.n) return;
    const uint32_t v = sorted_id(a, asc, i1);
    if (v >= a.V || sorted_id(a, asc, i1 - 1) != v || (b && sorted_id(a, asc, i0 - 1) == v)) return;
    if (tid < 64) {  // the last workgroup whose first entry is v's (the list is sorted): 64 probes at a time
        uint32_t lo = b + 1, hi = a.blocks;  // v's at lo, not at hi
        while (hi - lo > 1) {
            const uint32_t step = (hi - lo + 63) / 64, at = lo + (tid + 1) * step;
            const uint64_t in = __ballot(at < hi && sorted_id(a, asc, at * E) == v);
            const uint32_t k = __popcll(in);  // the probes that hold v come first
            hi = min(hi, lo + (k + 1) * step);
            lo += k * step;
        }
        if (tid == 0) s_last = lo;
    }
    __syncthreads();
    const uint32_t m = s_last - b, share = (m + NS - 1) / NS;
    const int64_t col = ((int64_t)blockIdx.y * L + ln) * VEC;
    const bool on = col < a.D;
    float acc[VEC] = {};
    if (on) {
        const uint32_t j0 = b + 1 + min(m, s * share), j1 = b + 1 + min(m, (s + 1) * share);
#pragma unroll 8
        for (uint32_t j = j0; j < j1; ++j) {
            const float* p = a.head + (int64_t)j * a.D + col;
#pragma unroll
            for (int c = 0; c < VEC; ++c) acc[c] += p[c];
        }
    }
    Vec<float, VEC> o;
#pragma unroll
    for (int c = 0; c < VEC; ++c) o.v[c] = acc[c];
    part[tid] = o;
    __syncthreads();
    if (s || !on) return;
    const float* p = a.tail + (int64_t)b * a.D + col;
#pragma unroll
    for (int c = 0; c < VEC; ++c) acc[c] += p[c];
    for (int q = 1; q < NS && (uint32_t)q * share < m; ++q) add_vec<float, VEC>(acc, part[q * L + ln]);
    put_row<VEC>(a, v, col, acc);
}

// ---------------------------------------------------------------------------------- launches

enum BwdForm { kFew, kTable, kRank, kRadix };

struct BwdPlan {
    BwdForm form;
    int lanes, passes, bits;
    uint32_t tiles, blocks, slabs, rows;
    size_t list_a, list_b, hist, total, ascend, head, tail, named, bytes;
};

static BwdPlan bwd_plan(int64_t V, int64_t n, int64_t D, int vec) {
    BwdPlan p{};
    const int64_t per_row = (D + vec - 1) / vec;
    p.lanes = 1;
    while (p.lanes < 64 && p.lanes < per_row) p.lanes <<= 1;
    const int64_t NS = 256 / p.lanes;
    p.slabs = (uint32_t)((per_row + p.lanes - 1) / p.lanes);
    size_t o = 0;
    auto take = [&](size_t b) {
        const size_t at = o;
        o += align256(b);
        return at;
    };
    p.form = n <= kFewMost ? kFew : V * vec <= kTableMost ? kTable : n <= kRankMost ? kRank : kRadix;
    if (p.form == kTable) {
        int64_t blocks = 512 / p.slabs;  // two per compute unit
        if (blocks < 1) blocks = 1;
        const int64_t step = 8 * NS, rows = (n + blocks - 1) / blocks;
        p.rows = (uint32_t)((rows + step - 1) / step * step);
        p.blocks = (uint32_t)((n + p.rows - 1) / p.rows);
        p.head = take((size_t)p.blocks * V * D * 4);
        p.named = take((size_t)p.blocks * V);
    } else if (p.form != kFew) {
        p.blocks = (uint32_t)((n + NS * kSumRun - 1) / (NS * kSumRun));
        p.list_a = take((size_t)n * 8);
        p.head = take((size_t)p.blocks * D * 4);
        p.tail = take((size_t)p.blocks * D * 4);
        if (p.form == kRadix) {
            int key_bits = 1;
            while ((V >> key_bits) != 0) ++key_bits;  // ids 0 .. V (V: no row)
            p.passes = (key_bits + kSortBits - 1) / kSortBits;
            p.bits = (key_bits + p.passes - 1) / p.passes;
            p.tiles = (uint32_t)((n + kSortTile - 1) / kSortTile);
            p.list_b = take((size_t)n * 8);
            p.hist = take(((size_t)p.tiles << p.bits) * 4);
            p.total = take((4ull << p.bits));
            p.ascend = take(((size_t)p.tiles + 1) * 4);
        }
    }
    p.bytes = o;
    return p;
}

// the zeros of a dense gradient, in `parts` launches
struct ZeroPlan {
    char* base = nullptr;
    int64_t units = 0;
    ZeroPart edges{};
    int parts = 1, next = 0;

    ZeroPlan() = default;
    ZeroPlan(void* dw, size_t bytes, int parts_) : parts(parts_) {
        char *p = static_cast<char*>(dw), *end = p + bytes;
        size_t before = (16 - (uintptr_t)p % 16) % 16;
        if (before > bytes) before = bytes;
        base = p + before;
        units = (end - base) / 16;
        edges.edge[0] = reinterpret_cast<uint16_t*>(p);
        edges.nedge[0] = (int)before / 2;
        edges.edge[1] = reinterpret_cast<uint16_t*>(base + units * 16);
        edges.nedge[1] = (int)((end - base) % 16) / 2;
    }
    // the next launch's part and its workgroups
    ZeroPart take(uint32_t& blocks) {
        blocks = 0;
        ZeroPart z{};
        if (!base) return z;
        if (next == 0) z = edges;
        const int64_t u0 = units * next / parts, u1 = units * (next + 1) / parts;
        z.p = reinterpret_cast<uint4*>(base) + u0;
        z.units = u1 - u0;
        blocks = (uint32_t)((z.units + kZeroUnits - 1) / kZeroUnits);
        if (next == 0 && blocks == 0) blocks = 1;
        ++next;
        return z;
    }
};

// sorts the ids: a.list, or a.ascend where they may turn out to be sorted
static void launch_sort(const BwdPlan& p, char* w, SumArgs& a, ZeroPlan zeros, hipStream_t s) {
    uint2 *la = reinterpret_cast<uint2*>(w + p.list_a), *lb = reinterpret_cast<uint2*>(w + p.list_b);
    uint32_t zb;
    if (p.form == kRank) {
        const uint32_t blocks = (a.n + 4 * kRankOwn - 1) / (4 * kRankOwn);
        const ZeroPart z = zeros.take(zb);
        hipLaunchKernelGGL(sort_rank_kernel, dim3(blocks + zb), dim3(256), 0, s, a.n, a.ids, a.V, la, blocks, z);
        a.list = la;
        return;
    }
    SortArgs t{};
    t.n = a.n;
    t.V = a.V;
    t.ids = a.ids;
    t.bits = p.bits;
    t.tiles = p.tiles;
    t.hist = reinterpret_cast<uint32_t*>(w + p.hist);
    t.total = reinterpret_cast<uint32_t*>(w + p.total);
    t.ascend = reinterpret_cast<uint32_t*>(w + p.ascend);
    const unsigned scan_blocks = ((1u << p.bits) + 63) / 64;
    for (int pass = 0; pass < p.passes; ++pass) {
        t.in = pass == 0 ? nullptr : pass & 1 ? la : lb;
        t.out = pass & 1 ? lb : la;
        t.shift = pass * p.bits;
        const ZeroPart z0 = zeros.take(zb);
        if (pass == 0) {
            hipLaunchKernelGGL((sort_count_kernel<true>), dim3(p.tiles + zb), dim3(256), 0, s, t, z0);
            hipLaunchKernelGGL((sort_scan_kernel<true>), dim3(scan_blocks + 1), dim3(1024), 0, s, t);
        } else {
            hipLaunchKernelGGL((sort_count_kernel<false>), dim3(p.tiles + zb), dim3(256), 0, s, t, z0);
            hipLaunchKernelGGL((sort_scan_kernel<false>), dim3(scan_blocks), dim3(1024), 0, s, t);
        }
        const ZeroPart z1 = zeros.take(zb);
        if (pass == 0)
            hipLaunchKernelGGL((sort_scatter_kernel<true>), dim3(p.tiles + zb), dim3(256), 0, s, t, z1);
        else
            hipLaunchKernelGGL((sort_scatter_kernel<false>), dim3(p.tiles + zb), dim3(256), 0, s, t, z1);
    }
    a.list = t.out;
    a.ascend = t.ascend;
}

template <typename GT, int VEC>
static void launch_sums(const BwdPlan& p, const SumArgs& a, uint32_t zero_blocks, hipStream_t s) {
    const dim3 block(256);
    switch (p.form) {
        case kFew:
            hipLaunchKernelGGL((embed_few_kernel<GT, VEC>), dim3(a.n + zero_blocks, p.slabs), block, 0, s, a);
            break;
        case kTable:
            hipLaunchKernelGGL((embed_table_kernel<GT, VEC>), dim3(a.blocks, p.slabs), block,
                               (size_t)a.V * 256 * VEC * sizeof(float), s, a);
            hipLaunchKernelGGL((embed_table_join_kernel<VEC>), dim3(a.V, p.slabs), block, 0, s, a);
            break;
        default:
            hipLaunchKernelGGL((embed_sum_kernel<GT, VEC>), dim3(a.blocks, p.slabs), block,
                               (2 * (256 / a.lanes) * kSumRun + 2) * sizeof(uint32_t), s, a);
            if (a.blocks > 1)
                hipLaunchKernelGGL((embed_join_kernel<VEC>), dim3(a.blocks, p.slabs), block, 0, s, a);
    }
}

template <typename GT>
static void launch_sums(int vec, const BwdPlan& p, const SumArgs& a, uint32_t zero_blocks, hipStream_t s) {
    switch (vec) {
        case 8: return launch_sums<GT, 8>(p, a, zero_blocks, s);
        case 4: return launch_sums<GT, 4>(p, a, zero_blocks, s);
        case 2: return launch_sums<GT, 2>(p, a, zero_blocks, s);
        default: return launch_sums<GT, 1>(p, a, zero_blocks, s);
    }
}

template <typename WT, typename OT, int VEC>
static void launch_fwd(int64_t V, int64_t n, int64_t D, const void* w, int64_t wstride, RowIds ids, float scale,
                       void* out, hipStream_t s) {
    const uint32_t per_row = (uint32_t)(D / VEC);
    const int64_t most = ((int64_t)1 << 30) / per_row;  // rows per launch: at most 2^30 pieces
    for (int64_t r0 = 0; r0 < n; r0 += most) {
        const uint32_t chunks = (uint32_t)((n - r0 < most ? n - r0 : most) * per_row);
        hipLaunchKernelGGL((embed_fwd_kernel<WT, OT, VEC>), dim3((chunks + 256 * kFwdPer - 1) / (256 * kFwdPer)), dim3(256), 0, s, chunks,
                           fast_div(per_row), (uint32_t)V, static_cast<const WT*>(w), wstride, ids, r0, scale,
                           static_cast<OT*>(out));
    }
}

template <typename WT, typename OT>
static void launch_fwd(int vec, int64_t V, int64_t n, int64_t D, const void* w, int64_t wstride, RowIds ids,
                       float scale, void* out, hipStream_t s) {
    switch (vec) {
        case 8: return launch_fwd<WT, OT, 8>(V, n, D, w, wstride, ids, scale, out, s);
        case 4: return launch_fwd<WT, OT, 4>(V, n, D, w, wstride, ids, scale, out, s);
        case 2: return launch_fwd<WT, OT, 2>(V, n, D, w, wstride, ids, scale, out, s);
        default: return launch_fwd<WT, OT, 1>(V, n, D, w, wstride, ids, scale, out, s);
    }
}

template <typename WT>
static void launch_fwd(int otype, int vec, int64_t V, int64_t n, int64_t D, const void* w, int64_t wstride, RowIds ids,
                       float scale, void* out, hipStream_t s) {
    if (otype == HGSR_F32) return launch_fwd<WT, float>(vec, V, n, D, w, wstride, ids, scale, out, s);
    if (otype == HGSR_F16) return launch_fwd<WT, f16_t>(vec, V, n, D, w, wstride, ids, scale, out, s);
    return launch_fwd<WT, bf16_t>(vec, V, n, D, w, wstride, ids, scale, out, s);
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
    int vec = vec_width(most, D, wstride, weight, elem_size(wtype));
    const int vo = vec_width(most, D, D, out, elem_size(otype));
    if (vo < vec) vec = vo;
    const RowIds id{ids, ids_stride, ids64};
    hipStream_t s = as_stream(stream);
    {
        KernelTimer kt("embed_fwd", s);
        if (wtype == HGSR_F32)
            launch_fwd<float>(otype, vec, V, n, D, weight, wstride, id, scale, out, s);
        else if (wtype == HGSR_F16)
            launch_fwd<f16_t>(otype, vec, V, n, D, weight, wstride, id, scale, out, s);
        else
            launch_fwd<bf16_t>(otype, vec, V, n, D, weight, wstride, id, scale, out, s);
    }
    return check_launch("embed_fwd");
}

extern "C" size_t hgsr_embed_bwd_ws_bytes(int64_t V, int64_t n, int64_t D) {
    if (V <= 0 || n <= 0 || D < 1) return 0;
    size_t most = 0;
    for (int vec = 1; vec <= 8; vec <<= 1) {  // the call picks the width by the tensors' alignment
        const size_t b = bwd_plan(V, n, D, vec).bytes;
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
    HGSR_REQUIRE(dw_bytes / (kZeroUnits * 16) < (1ull << 30), "embed_bwd: table too large");
    SumArgs a{};
    a.n = (uint32_t)n;
    a.V = (uint32_t)V;
    a.D = D;
    a.ids = RowIds{ids, ids_stride, ids64};
    a.g = g;
    a.gstride = gstride;
    a.dw = dw;
    a.dwstride = dwstride;
    a.dwtype = dwtype;
    a.accumulate = accumulate != 0;
    a.scale = scale;
    if (n == 0) {
        if (!accumulate) {
            uint32_t zb;
            ZeroPlan zeros(dw, dw_bytes, 1);
            const ZeroPart z = zeros.take(zb);
            hipLaunchKernelGGL(zero_kernel, dim3(zb), dim3(256), 0, s, z);
        }
        return check_launch("embed_bwd");
    }
    HGSR_REQUIRE(g && ids, "embed_bwd: null pointer");
    const int most = gtype == HGSR_F32 ? 4 : 8;
    int vec = vec_width(most, D, gstride, g, elem_size(gtype));
    const int vo = vec_width(most, D, dwstride, dw, elem_size(dwtype));
    if (vo < vec) vec = vo;
    const BwdPlan p = bwd_plan(V, n, D, vec);
    if (p.bytes > ws_bytes || (p.bytes && !ws)) {
        set_error("embed_bwd: workspace of %zu bytes, %zu needed", ws ? ws_bytes : (size_t)0, p.bytes);
        return HGSR_EWORKSPACE;
    }
    char* w = static_cast<char*>(ws);
    a.lanes = p.lanes;
    a.blocks = p.blocks;
    a.rows = p.rows;
    a.head = reinterpret_cast<float*>(w + p.head);
    a.tail = reinterpret_cast<float*>(w + p.tail);
    a.named = reinterpret_cast<uint8_t*>(w + p.named);
    KernelTimer kt("embed_bwd", s);
    uint32_t zero_blocks = 0;
    if (p.form == kFew && !accumulate) {  // about 32 KB of zeros per workgroup
        const int64_t rows = 32768 / ((int64_t)p.lanes * vec * elem_size(dwtype));
        a.rows = (uint32_t)(rows < 1 ? 1 : rows > kFewRows ? kFewRows : rows);
        zero_blocks = (uint32_t)((V + a.rows - 1) / a.rows);
    } else if (p.form == kRank || p.form == kRadix) {
        ZeroPlan zeros;
        if (!accumulate) zeros = ZeroPlan(dw, dw_bytes, p.form == kRank ? 1 : 2 * p.passes);
        launch_sort(p, w, a, zeros, s);
    }
    if (gtype == HGSR_F32)
        launch_sums<float>(vec, p, a, zero_blocks, s);
    else if (gtype == HGSR_F16)
        launch_sums<f16_t>(vec, p, a, zero_blocks, s);
    else
        launch_sums<bf16_t>(vec, p, a, zero_blocks, s);
    return check_launch("embed_bwd");
}
