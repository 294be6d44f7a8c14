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

template <typename WT, typename OT, int VEC>
__global__ __launch_bounds__(256) void embed_fwd_kernel(uint32_t chunks, FastDiv per_row, uint32_t V,
                                                        const WT* __restrict__ w, int64_t wstride, RowIds ids,
                                                        int64_t row0, float scale, OT* __restrict__ out) {
    const uint32_t c = blockIdx.x * 256 + threadIdx.x;
    if (c >= chunks) return;
    const uint32_t r = per_row.div(c), col = (c - r * per_row.d) * VEC;
    const int64_t row = row0 + r;
    const uint32_t id = ids.get(row, V);
    Vec<OT, VEC> o;
    if (id < V) {
        const Vec<WT, VEC> x = load_vec<WT, VEC>(w + (int64_t)id * wstride + col);
#pragma unroll
        for (int k = 0; k < VEC; ++k) o.v[k] = (OT)((float)x.v[k] * scale);
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) o.v[k] = (OT)0.0f;
    }
    store_vec<OT, VEC>(out + row * ((int64_t)per_row.d * VEC) + col, o);
}

// --------------------------------------------------------------------------- sort of (id, i)
// Least-significant-digit radix sort, digits of up to 11 bits: per pass the tiles' digit counts,
// their prefix over the tiles, and a stable scatter.
constexpr int kSortTile = 4096;  // entries per workgroup: 4 waves x 16 rounds x 64 lanes
constexpr int kSortBits = 11;

template <bool FIRST>
__device__ __forceinline__ uint2 sort_entry(const RowIds& ids, uint32_t V, const uint2* __restrict__ in, uint32_t i) {
    if (FIRST) return make_uint2(ids.get(i, V), i);
    return in[i];
}

// touched (nullable, first pass only): cleared here, set by the last pass's scatter
template <bool FIRST>
__global__ __launch_bounds__(256) void sort_count_kernel(uint32_t n, RowIds ids, uint32_t V,
                                                         const uint2* __restrict__ in, int shift, int bits,
                                                         uint32_t tiles, uint32_t* __restrict__ hist,
                                                         uint8_t* __restrict__ touched) {
    __shared__ uint32_t h[1 << kSortBits];
    const uint32_t bins = 1u << bits;
    for (uint32_t b = threadIdx.x; b < bins; b += 256) h[b] = 0;
    __syncthreads();
    const uint32_t base = blockIdx.x * kSortTile;
    for (int k = 0; k < kSortTile / 256; ++k) {
        const uint32_t i = base + k * 256 + threadIdx.x;
        if (i < n) atomicAdd(&h[(sort_entry<FIRST>(ids, V, in, i).x >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < bins; b += 256) hist[(size_t)b * tiles + blockIdx.x] = h[b];
    if (FIRST && touched)
        for (uint32_t v = blockIdx.x * 256 + threadIdx.x; v < V; v += gridDim.x * 256) touched[v] = 0;
}

// one wave per digit: exclusive prefix of its counts over the tiles, and their total
__global__ __launch_bounds__(256) void sort_scan_kernel(uint32_t bins, uint32_t tiles, uint32_t* __restrict__ hist,
                                                        uint32_t* __restrict__ total) {
    const uint32_t b = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (b >= bins) return;
    uint32_t* h = hist + (size_t)b * tiles;
    uint32_t carry = 0;
    for (uint32_t t0 = 0; t0 < tiles; t0 += 64) {
        const uint32_t t = t0 + lane, v = t < tiles ? h[t] : 0;
        uint32_t inc = v;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t o = __shfl_up(inc, d);
            if (lane >= d) inc += o;
        }
        if (t < tiles) h[t] = carry + inc - v;
        carry += __shfl(inc, 63);
    }
    if (lane == 0) total[b] = carry;
}

template <bool FIRST>
__global__ __launch_bounds__(256) void sort_scatter_kernel(uint32_t n, RowIds ids, uint32_t V,
                                                           const uint2* __restrict__ in, int shift, int bits,
                                                           uint32_t tiles, const uint32_t* __restrict__ hist,
                                                           const uint32_t* __restrict__ total,
                                                           uint2* __restrict__ out, uint8_t* __restrict__ touched) {
    constexpr int ROUNDS = kSortTile / 256;
    __shared__ uint32_t cnt[4][1 << kSortBits];  // per wave: count, then where its entries of the digit go
    __shared__ uint32_t wsum[4];
    const uint32_t bins = 1u << bits;
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
    for (uint32_t b = tid; b < 4 * bins; b += 256) cnt[b >> bits][b & (bins - 1)] = 0;
    __syncthreads();
    const uint32_t base = blockIdx.x * kSortTile + w * (kSortTile / 4);
    uint2 e[ROUNDS];
    uint32_t rank[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const uint32_t i = base + r * 64 + lane;
        if (i < n) e[r] = sort_entry<FIRST>(ids, V, in, i);
    }
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        // the lanes of this wave whose digit equals mine; the first of them adds their number
        const bool on = base + r * 64 + lane < n;
        const uint32_t d = on ? (e[r].x >> shift) & (bins - 1) : 0;
        uint64_t same = __ballot(on);
        if (!on) same = ~same;
        for (int k = 0; k < bits; ++k) {
            const uint64_t m = __ballot((d >> k) & 1);
            same &= (d >> k) & 1 ? m : ~m;
        }
        const int first = __ffsll((unsigned long long)same) - 1;
        uint32_t old = 0;
        if (on && lane == first) old = atomicAdd(&cnt[w][d], (uint32_t)__popcll(same));
        rank[r] = __shfl(old, first) + __popcll(same & ((1ull << lane) - 1));
    }
    __syncthreads();
    // digit b's entries of this tile start at (entries of smaller digits) + (its entries in earlier
    // tiles); 8 consecutive digits per thread
    constexpr int PER = (1 << kSortBits) / 256;
    uint32_t mine[PER], sum = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const uint32_t b = tid * PER + k;
        mine[k] = b < bins ? total[b] : 0;
        sum += mine[k];
    }
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
            uint32_t p = at + hist[(size_t)b * tiles + blockIdx.x];
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
    for (int r = 0; r < ROUNDS; ++r) {
        if (base + r * 64 + lane < n) {
            out[cnt[w][(e[r].x >> shift) & (bins - 1)] + rank[r]] = e[r];
            if (touched && e[r].x < V) touched[e[r].x] = 1;
        }
    }
}

// ------------------------------------------------------------------- sums of the sorted list
// A subgroup of `lanes` lanes holds VEC columns per lane and walks kSumRun consecutive entries;
// a workgroup's 256 / lanes subgroups take consecutive pieces.  Columns beyond lanes * VEC: grid.y.
constexpr int kSumRun = 16;

struct SumArgs {
    uint32_t n, V;
    int64_t D;
    const uint2* list;  // sorted (id, i)
    const void* g;
    int64_t gstride;
    void* dw;
    int64_t dwstride;
    int dwtype, accumulate;
    float scale;
    int lanes;          // lanes per subgroup, a power of two
    uint32_t blocks;    // workgroups over the list
    float *head, *tail;  // [blocks][D]: the sums of a workgroup's runs that began before it / go on after it
    const uint8_t* touched;
    uint32_t zero_rows;  // rows per zeroing workgroup
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

template <typename GT, int VEC>
__global__ __launch_bounds__(256) void embed_sum_kernel(const SumArgs a) {
    extern __shared__ uint32_t key[];         // [1 + E + 1]: the entry before, the workgroup's, the one after
    __shared__ Vec<float, VEC> part[2][256];  // [0]: run that began before the subgroup, [1]: goes on after it
    __shared__ int state[256];                // 1: has a part[0], 2: which goes on after it, 4: has a part[1]
    const int tid = threadIdx.x, L = a.lanes, s = tid / L, ln = tid & (L - 1), NS = 256 / L;
    const uint32_t E = NS * kSumRun;
    uint32_t* pos = key + E + 2;
    const int64_t col = ((int64_t)blockIdx.y * L + ln) * VEC;
    const bool on = col < a.D;
    if (blockIdx.x >= a.blocks) {  // rows that no id names
        const uint32_t r0 = (blockIdx.x - a.blocks) * a.zero_rows;
        float z[VEC] = {};
        for (uint32_t k = s; k < a.zero_rows; k += NS) {
            const uint32_t v = r0 + k;
            if (v < a.V && on && !a.touched[v]) put_row<VEC>(a, v, col, z);
        }
        return;
    }
    constexpr uint32_t NONE = ~0u;
    const uint32_t i0 = blockIdx.x * E;
    for (uint32_t k = tid; k < E; k += 256) {
        const uint32_t i = i0 + k;
        const uint2 e = i < a.n ? a.list[i] : make_uint2(NONE, 0);
        key[1 + k] = e.x;
        pos[k] = e.y;
    }
    if (tid == 0) {
        key[0] = i0 ? a.list[i0 - 1].x : NONE;
        key[1 + E] = i0 + E < a.n ? a.list[i0 + E].x : NONE;
    }
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
#pragma unroll
            for (int c = 0; c < VEC; ++c) acc[c] += (float)x[u].v[c];
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
    auto add = [&](int sub) {
        const Vec<float, VEC> p = part[0][sub * L + ln];
#pragma unroll
        for (int c = 0; c < VEC; ++c) acc[c] += p.v[c];
    };
    auto keep = [&](float* to) {
        float* p = to + (int64_t)blockIdx.x * a.D + col;
#pragma unroll
        for (int c = 0; c < VEC; ++c) p[c] = acc[c];
    };
    if (!on) return;
    if (st & 4) {  // a run that begins here and goes on: its owner adds the later subgroups' shares
        const Vec<float, VEC> p = part[1][tid];
#pragma unroll
        for (int c = 0; c < VEC; ++c) acc[c] = p.v[c];
        int q = s + 1;
        bool open = true;
        for (; q < NS && open; ++q) {
            add(q);
            open = state[q] & 2;
        }
        if (open)
            keep(a.tail);
        else
            put_row<VEC>(a, key[e0 + kSumRun], col, acc);
    }
    if (s == 0 && (st & 1)) {  // the run that an earlier workgroup began
#pragma unroll
        for (int c = 0; c < VEC; ++c) acc[c] = 0.0f;
        add(0);
        for (int q = 1; q < NS && (state[q - 1] & 2); ++q) add(q);
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
    const uint32_t E = NS * kSumRun, b = blockIdx.x, i0 = b * E, i1 = i0 + E;
    if (i1 >= a.n) return;
    const uint32_t v = a.list[i1].x;
    if (v >= a.V || a.list[i1 - 1].x != v || (b && a.list[i0 - 1].x == v)) return;
    if (tid == 0) {  // the last workgroup whose first entry is v's (the list is sorted)
        uint32_t lo = b + 1, hi = a.blocks - 1;
        while (lo < hi) {
            const uint32_t mid = hi - ((hi - lo) >> 1);
            if (a.list[mid * E].x == v)
                lo = mid;
            else
                hi = mid - 1;
        }
        s_last = lo;
    }
    __syncthreads();
    const uint32_t m = s_last - b, share = (m + NS - 1) / NS;
    const int64_t col = ((int64_t)blockIdx.y * L + ln) * VEC;
    const bool on = col < a.D;
    float acc[VEC] = {};
    if (on) {
        const uint32_t j0 = b + 1 + min(m, s * share), j1 = b + 1 + min(m, (s + 1) * share);
#pragma unroll 4
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
    for (int q = 1; q < NS && (uint32_t)q * share < m; ++q) {
        const Vec<float, VEC> x = part[q * L + ln];
#pragma unroll
        for (int c = 0; c < VEC; ++c) acc[c] += x.v[c];
    }
    put_row<VEC>(a, v, col, acc);
}

__global__ __launch_bounds__(256) void zero_rows_kernel(SumArgs a) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)a.V * a.D) return;
    const float z[1] = {0.0f};
    put_row<1>(a, (uint32_t)(i / a.D), i % a.D, z);
}

// ---------------------------------------------------------------------------------- launches

struct BwdPlan {
    int vec, lanes, passes, bits;
    uint32_t tiles, blocks, slabs;
    size_t list_a, list_b, hist, total, touched, head, tail, bytes;
};

// vec: columns per lane; the workspace query takes 1, where a list piece is shortest
static BwdPlan bwd_plan(int64_t V, int64_t n, int64_t D, int vec) {
    BwdPlan p{};
    p.vec = vec;
    const int64_t per_row = (D + vec - 1) / vec;
    p.lanes = 1;
    while (p.lanes < 64 && p.lanes < per_row) p.lanes <<= 1;
    const int64_t E = (int64_t)(256 / p.lanes) * kSumRun;
    p.blocks = (uint32_t)((n + E - 1) / E);
    p.slabs = (uint32_t)((per_row + p.lanes - 1) / p.lanes);
    int key_bits = 1;
    while ((V >> key_bits) != 0) ++key_bits;  // ids 0 .. V (V: no row)
    p.passes = (key_bits + kSortBits - 1) / kSortBits;
    p.bits = (key_bits + p.passes - 1) / p.passes;
    p.tiles = (uint32_t)((n + kSortTile - 1) / kSortTile);
    size_t o = 0;
    auto take = [&](size_t b) {
        const size_t at = o;
        o += align256(b);
        return at;
    };
    p.list_a = take((size_t)n * 8);
    p.list_b = take((size_t)n * 8);
    p.hist = take(((size_t)p.tiles << p.bits) * 4);
    p.total = take((4ull << p.bits));
    p.touched = take((size_t)V);
    p.head = take((size_t)p.blocks * D * 4);
    p.tail = take((size_t)p.blocks * D * 4);
    p.bytes = o;
    return p;
}

template <typename GT, int VEC>
static void launch_sums(const SumArgs& a, uint32_t zero_blocks, uint32_t slabs, hipStream_t s) {
    hipLaunchKernelGGL((embed_sum_kernel<GT, VEC>), dim3(a.blocks + zero_blocks, slabs), dim3(256),
                       (2 * (256 / a.lanes) * kSumRun + 2) * sizeof(uint32_t), s, a);
    if (a.blocks > 1) hipLaunchKernelGGL((embed_join_kernel<VEC>), dim3(a.blocks, slabs), dim3(256), 0, s, a);
}

template <typename GT>
static void launch_sums(int vec, const SumArgs& a, uint32_t zero_blocks, uint32_t slabs, hipStream_t s) {
    switch (vec) {
        case 8: return launch_sums<GT, 8>(a, zero_blocks, slabs, s);
        case 4: return launch_sums<GT, 4>(a, zero_blocks, slabs, s);
        case 2: return launch_sums<GT, 2>(a, zero_blocks, slabs, s);
        default: return launch_sums<GT, 1>(a, zero_blocks, slabs, s);
    }
}

template <typename WT, typename OT, int VEC>
static void launch_fwd(int64_t V, int64_t n, int64_t D, const void* w, int64_t wstride, RowIds ids, float scale,
                       void* out, hipStream_t s) {
    const uint32_t per_row = (uint32_t)(D / VEC);
    const int64_t most = ((int64_t)1 << 30) / per_row;  // rows per launch: at most 2^30 pieces
    for (int64_t r0 = 0; r0 < n; r0 += most) {
        const uint32_t chunks = (uint32_t)((n - r0 < most ? n - r0 : most) * per_row);
        hipLaunchKernelGGL((embed_fwd_kernel<WT, OT, VEC>), dim3((chunks + 255) / 256), dim3(256), 0, s, chunks,
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
    HGSR_REQUIRE(n >= 0 && n < (1ll << 31) - kSortTile, "%s: %lld ids: at most 2^31 - 4097", what, (long long)n);
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
    if (V < 0 || n <= 0 || D < 1) return 0;
    return bwd_plan(V, n, D, 1).bytes;
}

extern "C" int hgsr_embed_bwd(int64_t V, int64_t n, int64_t D, const void* g, int gtype, int64_t gstride,
                              const void* ids, int ids64, int64_t ids_stride, float scale, void* dw, int dwtype,
                              int64_t dwstride, int accumulate, void* ws, size_t ws_bytes, hgsr_stream_t stream) {
    if (int st = check_dims("embed_bwd", V, n, D)) return st;
    HGSR_REQUIRE(type_ok(gtype) && type_ok(dwtype), "embed_bwd: unknown element type");
    HGSR_REQUIRE(gstride >= 0 && dwstride >= D && ids_stride >= 0, "embed_bwd: bad stride");
    if (V == 0) return HGSR_OK;
    HGSR_REQUIRE(dw, "embed_bwd: null pointer");
    hipStream_t s = as_stream(stream);
    SumArgs a{};
    a.n = (uint32_t)n;
    a.V = (uint32_t)V;
    a.D = D;
    a.g = g;
    a.gstride = gstride;
    a.dw = dw;
    a.dwstride = dwstride;
    a.dwtype = dwtype;
    a.accumulate = accumulate != 0;
    a.scale = scale;
    if (n == 0) {
        if (!accumulate) {
            const int64_t blocks = (V * D + 255) / 256;
            HGSR_REQUIRE(blocks < (1ll << 31), "embed_bwd: table too large");
            hipLaunchKernelGGL(zero_rows_kernel, dim3((unsigned)blocks), dim3(256), 0, s, a);
        }
        return check_launch("embed_bwd");
    }
    HGSR_REQUIRE(g && ids && ws, "embed_bwd: null pointer");
    const int most = gtype == HGSR_F32 ? 4 : 8;
    int vec = vec_width(most, D, gstride, g, elem_size(gtype));
    const int vo = vec_width(most, D, dwstride, dw, elem_size(dwtype));
    if (vo < vec) vec = vo;
    const BwdPlan p = bwd_plan(V, n, D, vec);
    if (p.bytes > ws_bytes) {
        set_error("embed_bwd: workspace of %zu bytes, %zu needed", ws_bytes, p.bytes);
        return HGSR_EWORKSPACE;
    }
    char* w = static_cast<char*>(ws);
    uint2 *in = reinterpret_cast<uint2*>(w + p.list_a), *out = reinterpret_cast<uint2*>(w + p.list_b);
    uint32_t *hist = reinterpret_cast<uint32_t*>(w + p.hist), *total = reinterpret_cast<uint32_t*>(w + p.total);
    uint8_t* touched = accumulate ? nullptr : reinterpret_cast<uint8_t*>(w + p.touched);
    const RowIds id{ids, ids_stride, ids64};
    KernelTimer kt("embed_bwd", s);
    for (int pass = 0; pass < p.passes; ++pass) {
        const int shift = pass * p.bits;
        uint8_t* set = pass == p.passes - 1 ? touched : nullptr;
        if (pass == 0)
            hipLaunchKernelGGL((sort_count_kernel<true>), dim3(p.tiles), dim3(256), 0, s, a.n, id, a.V, in, shift, p.bits,
                               p.tiles, hist, touched);
        else
            hipLaunchKernelGGL((sort_count_kernel<false>), dim3(p.tiles), dim3(256), 0, s, a.n, id, a.V, in, shift,
                               p.bits, p.tiles, hist, nullptr);
        hipLaunchKernelGGL(sort_scan_kernel, dim3(((1u << p.bits) + 3) / 4), dim3(256), 0, s, 1u << p.bits, p.tiles,
                           hist, total);
        if (pass == 0)
            hipLaunchKernelGGL((sort_scatter_kernel<true>), dim3(p.tiles), dim3(256), 0, s, a.n, id, a.V, in, shift,
                               p.bits, p.tiles, hist, total, out, set);
        else
            hipLaunchKernelGGL((sort_scatter_kernel<false>), dim3(p.tiles), dim3(256), 0, s, a.n, id, a.V, in, shift,
                               p.bits, p.tiles, hist, total, out, set);
        uint2* t = in;
        in = out;
        out = t;
    }
    a.list = in;
    a.lanes = p.lanes;
    a.blocks = p.blocks;
    a.head = reinterpret_cast<float*>(w + p.head);
    a.tail = reinterpret_cast<float*>(w + p.tail);
    a.touched = touched;
    uint32_t zero_blocks = 0;
    if (!accumulate) {  // about 32 KB of zeros per workgroup
        const int64_t rows = 32768 / ((int64_t)p.lanes * vec * elem_size(dwtype));
        a.zero_rows = (uint32_t)(rows < 1 ? 1 : rows);
        zero_blocks = (uint32_t)((V + a.zero_rows - 1) / a.zero_rows);
    }
    if (gtype == HGSR_F32)
        launch_sums<float>(vec, a, zero_blocks, p.slabs, s);
    else if (gtype == HGSR_F16)
        launch_sums<f16_t>(vec, a, zero_blocks, p.slabs, s);
    else
        launch_sums<bf16_t>(vec, a, zero_blocks, p.slabs, s);
    return check_launch("embed_bwd");
}
