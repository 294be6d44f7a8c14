// K19: a cache of rows held in 8 bits -- quantised as they are written into their slots, and read
// back by slot (the anchor features of a merged scene, or any rows kept for later reads).
//
//   write  s = max(max |x| over a group of columns * (1 / top), 2^-100),  code = round(x / s)
//   read   x' = code * s
//
// Both are bound by memory: a write's lane moves 16 consecutive columns of a row, a read's what fills
// 16 bytes of its output; the lanes of a group find its maximum among themselves.  500k rows of 32
// floats, every other slot of a million: the write 24.5 us in its three launches (84 MB, 3.4 TB/s; the
// slots' lines are stored in part), the read 16.2 (5.2 TB/s); 16k rows of 2048 read to bf16: 16.4 us
// (6.0 TB/s).
#include "rows.h"

namespace hgsr {

constexpr float kScaleFloor = 0x1p-100f;

template <typename I>
struct CacheArgs {
    uint32_t capacity, chunks;         // chunks: lanes' pieces of this launch
    FastDiv per_row;
    int64_t row0, n;
    uint32_t D;
    int group, glog;                   // group = 1 << glog columns
    uint8_t* codes;
    float* scales;
    int64_t cstride, sstride;
    RowIds<I> slots;                   // slots.p == nullptr: slot i
    void* x;                           // rows written, or the rows that a read fills
    int64_t xstride;
    const int32_t* last;               // write: the last row of each named slot (nullable), unless
    const uint32_t* distinct;          // this is set: no slot is named twice
    int tlog;                          // write of few rows: the table has 1 << tlog places
};

template <typename I>
__device__ __forceinline__ uint32_t slot_of(const CacheArgs<I>& a, int64_t i) {
    if (!a.slots.p) return i < (int64_t)a.capacity ? (uint32_t)i : a.capacity;
    return a.slots.get(i, a.capacity);
}

// x / s as a float whose last bit stands for what lies below it ("round to odd"): any later
// rounding to fewer bits gives what rounding the exact quotient would.  inv = 1 / s, s a normal
// float; q is within one step of the quotient after its correction, and the remainder x - q s of
// such a q is exact in one fused operation.
__device__ __forceinline__ float quotient_odd(float x, float s, float inv) {
#pragma clang fp contract(off)
    float q = x * inv;
    q = __builtin_fmaf(__builtin_fmaf(-q, s, x), inv, q);
    const float r = __builtin_fmaf(-q, s, x);
    const uint32_t b = __float_as_uint(q);
    if (r != 0.0f && q != 0.0f && !(b & 1)) return __uint_as_float((r > 0.0f) == (q > 0.0f) ? b + 1 : b - 1);
    return q;
}

// The codes of VEC values of a group, four to a word.  The rounding of x / s is that of the exact
// quotient: q = x * (1 / s) is off by at most 2^-23 of it, so its rounding is the quotient's unless q lies
// that near to the border of two codes (5 of 100,000 int8 values, 1 of 100,000 e4m3 ones); a wave that
// holds such a value divides exactly.  16-bit rows are bound by this arithmetic: 16k x 2048 bf16 take
// 37 us with a comparison for every value and separate conversions.
template <int FMT, int VEC>
__device__ __forceinline__ void encode(const float* x, float s, float inv, uint32_t* w) {
#pragma clang fp contract(off)
    if (FMT == HGSR_INT8) {
        // q + 1.5 2^23 rounds q to a whole number and holds it in its low bits; |q| <= 127: q is off by
        // at most 2^-16
        constexpr float kWhole = 12582912.0f;
        uint32_t t[VEC];
        float off = 0.0f;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            const float q = x[k] * inv, r = q + kWhole;
            off = fmaxf(off, fabsf(q - (r - kWhole)));
            t[k] = __float_as_uint(r);
        }
        if (__any(off > 0.5f - 0x1p-15f)) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) t[k] = __float_as_uint(rintf(quotient_odd(x[k], s, inv)) + kWhole);
        }
#pragma unroll
        for (int k = 0; k < VEC; k += 4)
            w[k / 4] = __builtin_amdgcn_perm(t[k + 1], t[k], 0x0c0c0400u) |
                       __builtin_amdgcn_perm(t[k + 3], t[k + 2], 0x04000c0cu);
        return;
    }
    // near: how far the mantissa's 20 bits behind the code's three are from the border, 0x80000; low: the
    // smallest magnitude but 0 (below 2^-6 codes have fewer bits)
    float y[VEC];
    uint32_t near = ~0u, low = ~0u;
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
        y[k] = x[k] * inv;
        const uint32_t b = __float_as_uint(y[k]);
        near = min(near, (b - 0x7fffcu) & 0xfffffu);
        low = min(low, (b & 0x7fffffffu) - 1u);
    }
    if (__any(near <= 8u || low < 0x3c800000u - 1u)) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) y[k] = quotient_odd(x[k], s, inv);
    }
#pragma unroll
    for (int k = 0; k < VEC; k += 4) {
        const int v = __builtin_amdgcn_cvt_pk_fp8_f32(y[k], y[k + 1], 0, false);
        w[k / 4] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[k + 2], y[k + 3], v, true);
    }
}
template <int FMT>
__device__ __forceinline__ void decode4(uint32_t w, float* o) {
    if (FMT == HGSR_INT8) {
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = (float)(int8_t)(w >> (8 * k));
    } else {
        o[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0);
        o[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1);
        o[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2);
        o[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
    }
}

// ------------------------------------------------------------------------------------- write

// Few rows: no launch before the write, each of whose workgroups (4,096 columns) spends the time of n
// inserts.  2,048 rows of 1024 bf16 9 us, 16 with the launches below; of 2048 9.4 and 16.3; of 4096 17.2
// and 17.1; of 8192 30 and 23.
constexpr int kFewSlots = 2048;
constexpr int64_t kFewWork = 1ll << 33;  // n n D

static bool few_slots(int64_t n, int64_t D) { return n <= kFewSlots && n * n * D <= kFewWork; }

// More: `last` is the last row that names each slot.  Slots in strictly ascending order (a compacted
// index, a chunk appended) cannot repeat: the first launch finds out tile by tile, the second ends at once,
// and the write does not look.  Otherwise `last`, cleared by the first launch where rows name it, is raised
// to their numbers by the second: by an atomic for every row (500k rows of 32 floats into a million slots
// 58 us in all, 24 in order), or, up to 16,384 slots, of which each may have many rows, by tiles of rows in
// LDS first (270k rows of 12 into 404: 16 us, 105 by atomics).
constexpr int kSlotTile = 1024;
constexpr int kFewCapacity = 16384;
constexpr int kSlotWide = 16384;  // rows per workgroup and turn of the LDS form
// Every workgroup of the second launch reads all tiles' verdicts, so its grid does not grow with the rows: at
// most kSlotTile workgroups read no more verdicts than there are rows.
constexpr uint32_t kSlotBlocks = kSlotTile, kSlotWideBlocks = 256;

struct SlotWork {
    uint32_t* distinct;  // [1 + tiles]: the verdict, then the tiles' own
    int32_t* last;       // [capacity]
    uint32_t tiles;
};

template <typename I>
__global__ __launch_bounds__(256) void slot_check_kernel(uint32_t n, RowIds<I> slots, uint32_t capacity, SlotWork w) {
    __shared__ uint32_t s[kSlotTile + 1];
    const uint32_t base = blockIdx.x * kSlotTile;
    uint32_t c[kSlotTile / 256];
#pragma unroll
    for (int k = 0; k < kSlotTile / 256; ++k) {
        const uint32_t i = base + k * 256 + threadIdx.x;
        c[k] = i < n ? slots.get(i, capacity) : ~0u;
    }
    const uint32_t end = base + kSlotTile;
    if (threadIdx.x == 0) s[kSlotTile] = end < n ? slots.get(end, capacity) : ~0u;
#pragma unroll
    for (int k = 0; k < kSlotTile / 256; ++k) {
        s[k * 256 + threadIdx.x] = c[k];
        if (c[k] < capacity) w.last[c[k]] = -1;
    }
    __syncthreads();
    int up = 1;
#pragma unroll
    for (int k = 0; k < kSlotTile / 256; ++k) up &= c[k] < s[k * 256 + threadIdx.x + 1] || c[k] == ~0u;
    up = __syncthreads_and(up);
    if (threadIdx.x == 0) w.distinct[1 + blockIdx.x] = up;
}

// the tiles' verdicts joined; every thread of every workgroup of the second launch calls it
__device__ __forceinline__ bool slots_distinct(const SlotWork& w) {
    int up = 1;
    for (uint32_t t = threadIdx.x; t < w.tiles; t += blockDim.x) up &= w.distinct[1 + t];
    up = __syncthreads_and(up);
    if (blockIdx.x == 0 && threadIdx.x == 0) w.distinct[0] = up;
    return up;
}

template <typename I>
__global__ __launch_bounds__(1024) void slot_last_few_kernel(uint32_t n, RowIds<I> slots, uint32_t capacity, SlotWork w) {
    __shared__ int32_t last[kFewCapacity];
    if (slots_distinct(w)) return;
    for (uint32_t s = threadIdx.x; s < capacity; s += 1024) last[s] = -1;
    for (uint32_t base = blockIdx.x * kSlotWide;; base += gridDim.x * kSlotWide) {
        const uint32_t i0 = base + threadIdx.x;
        uint32_t c[kSlotWide / 1024];
#pragma unroll
        for (int k = 0; k < kSlotWide / 1024; ++k)
            c[k] = i0 + k * 1024 < n ? slots.get(i0 + k * 1024, capacity) : capacity;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kSlotWide / 1024; ++k)
            if (c[k] < capacity) atomicMax(&last[c[k]], (int32_t)(i0 + k * 1024));
        if (n - base <= gridDim.x * kSlotWide) break;
    }
    __syncthreads();
    for (uint32_t s = threadIdx.x; s < capacity; s += 1024)
        if (last[s] >= 0) atomicMax(&w.last[s], last[s]);
}

template <typename I>
__global__ __launch_bounds__(256) void slot_last_each_kernel(uint32_t n, RowIds<I> slots, uint32_t capacity, SlotWork w) {
    if (slots_distinct(w)) return;
    for (uint32_t t = blockIdx.x; t < w.tiles; t += gridDim.x) {
#pragma unroll
        for (int k = 0; k < kSlotTile / 256; ++k) {
            const uint32_t i = t * kSlotTile + k * 256 + threadIdx.x, c = i < n ? slots.get(i, capacity) : capacity;
            if (c < capacity) atomicMax(&w.last[c], (int32_t)i);
        }
    }
}

// VEC consecutive columns per lane, fewer where the row ends.  FEW: every workgroup finds the last row of
// each slot itself, in a table in LDS with at least twice as many places as rows (a slot lies at the first
// place from its hash on that no other slot holds).
template <typename XT, typename I, int FMT, int VEC, bool FEW>
__global__ __launch_bounds__(256) void rowcache_write_kernel(const CacheArgs<I> a) {
    __shared__ uint32_t key[FEW ? 2 * kFewSlots : 1];
    __shared__ int32_t last[FEW ? 2 * kFewSlots : 1];
    // An XCD's workgroups take consecutive rows, so that narrow rows' slots in order share its L2's lines
    // (500k rows of 32 floats 24.5 us, 25.3 without); wide rows share none and take as long either way (16k of
    // 2048 bf16 33.3 and 33.4 us, in order 27.6 and 28.1).
    const uint32_t c = xcd_remap(blockIdx.x, gridDim.x) * 256 + threadIdx.x;
    const bool in = c < a.chunks;
    const uint32_t r = a.per_row.div(in ? c : 0);
    const int64_t row = a.row0 + r;
    const uint32_t D = a.D, col = in ? (c - r * a.per_row.d) * VEC : D;
    const uint32_t slot = slot_of(a, row);
    float x[VEC];
    const XT* p = static_cast<const XT*>(a.x) + row * a.xstride + col;
    if (col + VEC <= D) {
        const Vec<XT, VEC> v = load_vec<XT, VEC>(p);
#pragma unroll
        for (int k = 0; k < VEC; ++k) x[k] = (float)v.v[k];
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) x[k] = col + k < D ? (float)p[k] : 0.0f;
    }
    bool on = col < D && slot < a.capacity;
    if (FEW) {
        constexpr uint32_t NONE = ~0u;
        const uint32_t mask = (1u << a.tlog) - 1;
        const auto home = [&](uint32_t v) { return (v * 0x9e3779b9u) >> (32 - a.tlog); };
        for (uint32_t k = threadIdx.x; k <= mask; k += 256) {
            key[k] = NONE;
            last[k] = -1;
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < (uint32_t)a.n; i += 256) {
            const uint32_t v = slot_of(a, i);
            if (v >= a.capacity) continue;
            uint32_t h = home(v);
            for (;;) {
                const uint32_t old = atomicCAS(&key[h], NONE, v);
                if (old == NONE || old == v) break;
                h = (h + 1) & mask;
            }
            atomicMax(&last[h], (int32_t)i);
        }
        __syncthreads();
        if (on) {
            uint32_t h = home(slot);
            while (key[h] != slot) h = (h + 1) & mask;
            on = last[h] == (int32_t)row;
        }
    } else if (a.last && !*a.distinct && on) {
        on = a.last[slot] == (int32_t)row;
    }
    // the largest magnitude of the group as bits: infinities and NaN lie above every number
    const int lanes = a.group / VEC;  // a power of two, <= 8
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < VEC; ++k) m = max(m, __float_as_uint(x[k]) & 0x7fffffffu);
    for (int d = 1; d < lanes; d <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
    if (!on) return;
    const bool finite = m < 0x7f800000u;
    const float per = FMT == HGSR_INT8 ? 1.0f / 127.0f : 1.0f / 448.0f;
    const float s = fmaxf(__uint_as_float(m) * per, kScaleFloor), inv = 1.0f / s;
    uint32_t w[VEC / 4];
    encode<FMT, VEC>(x, s, inv, w);
#pragma unroll
    for (int k = 0; k < VEC / 4; ++k) w[k] = finite ? w[k] : 0u;
    uint8_t* to = a.codes + (int64_t)slot * a.cstride + col;
    if (col + VEC <= D) {
        Vec<uint8_t, VEC> o;
#pragma unroll
        for (int k = 0; k < VEC / 4; ++k) __builtin_memcpy(o.v + 4 * k, w + k, 4);
        store_vec<uint8_t, VEC>(to, o);
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            if (col + k < D) to[k] = (uint8_t)(w[k / 4] >> (8 * (k & 3)));
    }
    if ((col & (a.group - 1)) == 0)
        a.scales[(int64_t)slot * a.sstride + (col >> a.glog)] = finite ? s : __builtin_nanf("");
}

// -------------------------------------------------------------------------------------- read

// STREAM: the rows are stored past the caches.  WHOLE: no row ends inside a lane's piece.
template <typename OT, typename I, int FMT, int VEC, bool WHOLE, bool STREAM>
__global__ __launch_bounds__(256) void rowcache_read_kernel(const CacheArgs<I> a) {
    const uint32_t c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.chunks) return;
    const uint32_t r = a.per_row.div(c);
    const int64_t row = a.row0 + r;
    const uint32_t D = a.D, col = (c - r * a.per_row.d) * VEC;
    const uint32_t slot = slot_of(a, row);
    float x[VEC] = {};
    if (slot < a.capacity) {
        const uint8_t* p = a.codes + (int64_t)slot * a.cstride + col;
        const float s = a.scales[(int64_t)slot * a.sstride + (col >> a.glog)];
        uint32_t w[VEC / 4];
        if (WHOLE || col + VEC <= D) {
            const Vec<uint8_t, VEC> v = load_vec<uint8_t, VEC>(p);
#pragma unroll
            for (int k = 0; k < VEC / 4; ++k) __builtin_memcpy(w + k, v.v + 4 * k, 4);
        } else {
#pragma unroll
            for (int k = 0; k < VEC / 4; ++k) w[k] = 0;
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                if (col + k < D) w[k / 4] |= (uint32_t)p[k] << (8 * (k & 3));
        }
#pragma unroll
        for (int k = 0; k < VEC; k += 4) decode4<FMT>(w[k / 4], x + k);
#pragma unroll
        for (int k = 0; k < VEC; ++k) x[k] *= s;
    }
    OT* to = static_cast<OT*>(a.x) + row * D + col;
    if (WHOLE || col + VEC <= D) {
        Vec<OT, VEC> o;
#pragma unroll
        for (int k = 0; k < VEC; ++k) o.v[k] = (OT)x[k];
        if (STREAM)
            stream_vec<OT, VEC>(to, o);
        else
            store_vec<OT, VEC>(to, o);
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            if (col + k < D) to[k] = (OT)x[k];
    }
}

// ---------------------------------------------------------------------------------- launches

template <bool WRITE, typename T, int FMT, int VEC, typename I>
static void launch(const CacheArgs<I>& a, hipStream_t s) {
    const dim3 block(256), grid((a.chunks + 255) / 256);
    if constexpr (WRITE) {
        if (a.slots.p && a.n > 1 && few_slots(a.n, a.D))
            hipLaunchKernelGGL((rowcache_write_kernel<T, I, FMT, VEC, true>), grid, block, 0, s, a);
        else
            hipLaunchKernelGGL((rowcache_write_kernel<T, I, FMT, VEC, false>), grid, block, 0, s, a);
    } else {
        if (a.D % VEC)
            hipLaunchKernelGGL((rowcache_read_kernel<T, I, FMT, VEC, false, false>), grid, block, 0, s, a);
        else if (stream_out(a.n * (int64_t)a.D * (int64_t)sizeof(T)))
            hipLaunchKernelGGL((rowcache_read_kernel<T, I, FMT, VEC, true, true>), grid, block, 0, s, a);
        else
            hipLaunchKernelGGL((rowcache_read_kernel<T, I, FMT, VEC, true, false>), grid, block, 0, s, a);
    }
}

template <bool WRITE, typename T, int VEC, typename I>
static void launch(int format, CacheArgs<I> a, hipStream_t s) {
    // a write's rows are whole groups of lanes, so that no group crosses a wave
    const int64_t pieces = ((int64_t)a.D + VEC - 1) / VEC, groups = ((int64_t)a.D + a.group - 1) / a.group;
    const int64_t per_row = WRITE ? groups * (a.group / VEC) : pieces;
    const int64_t most = ((int64_t)1 << 30) / per_row;
    a.per_row = fast_div((uint32_t)per_row);
    for (a.row0 = 0; a.row0 < a.n; a.row0 += most) {
        a.chunks = (uint32_t)((a.n - a.row0 < most ? a.n - a.row0 : most) * per_row);
        if (format == HGSR_INT8)
            launch<WRITE, T, HGSR_INT8, VEC>(a, s);
        else
            launch<WRITE, T, HGSR_E4M3, VEC>(a, s);
    }
}

// the call's arguments that no kernel template hangs on
struct CacheCall {
    int64_t capacity, n, D, cstride, sstride, slots_stride, xstride;
    int group, format, type, slots64;
    const void* slots;
    void *codes, *x, *ws;
    float* scales;
};

static SlotWork slot_work(void* ws, int64_t n) {
    SlotWork w;
    w.tiles = (uint32_t)((n + kSlotTile - 1) / kSlotTile);
    w.distinct = static_cast<uint32_t*>(ws);
    w.last = reinterpret_cast<int32_t*>(static_cast<char*>(ws) + align256(((size_t)w.tiles + 1) * 4));
    return w;
}

template <bool WRITE, typename I>
static void launch(const CacheCall& c, hipStream_t s) {
    CacheArgs<I> a{};
    a.capacity = (uint32_t)c.capacity;
    a.n = c.n;
    a.D = (uint32_t)c.D;
    a.group = c.group;
    a.glog = c.group == 16 ? 4 : c.group == 32 ? 5 : c.group == 64 ? 6 : 7;
    a.codes = static_cast<uint8_t*>(c.codes);
    a.scales = c.scales;
    a.cstride = c.cstride;
    a.sstride = c.sstride;
    a.slots = RowIds<I>{static_cast<const I*>(c.slots), c.slots_stride};
    a.x = c.x;
    a.xstride = c.xstride;
    while ((1ll << a.tlog) < 2 * c.n && a.tlog < 30) ++a.tlog;
    if (WRITE && c.slots && !few_slots(c.n, c.D)) {
        const SlotWork w = slot_work(c.ws, c.n);
        const uint32_t n = (uint32_t)c.n, cap = a.capacity;
        hipLaunchKernelGGL((slot_check_kernel<I>), dim3(w.tiles), dim3(256), 0, s, n, a.slots, cap, w);
        const uint32_t wide = (n + kSlotWide - 1) / kSlotWide;
        if (cap <= kFewCapacity)
            hipLaunchKernelGGL((slot_last_few_kernel<I>), dim3(wide < kSlotWideBlocks ? wide : kSlotWideBlocks), dim3(1024),
                               0, s, n, a.slots, cap, w);
        else
            hipLaunchKernelGGL((slot_last_each_kernel<I>), dim3(w.tiles < kSlotBlocks ? w.tiles : kSlotBlocks), dim3(256), 0,
                               s, n, a.slots, cap, w);
        a.last = w.last;
        a.distinct = w.distinct;
    }
    // Columns per lane: a write 16, the smallest group (16k rows of 2048 bf16 in any order 34 us, 38 with
    // 8); a read what makes its stores 16 bytes (500k rows of 32 floats 16.2 us; 18.6 with 8 columns, whose
    // two stores are 32 bytes apart).
    if (c.type == HGSR_F32)
        launch<WRITE, float, WRITE ? 16 : 4>(c.format, a, s);
    else if (c.type == HGSR_F16)
        launch<WRITE, f16_t, WRITE ? 16 : 8>(c.format, a, s);
    else
        launch<WRITE, bf16_t, WRITE ? 16 : 8>(c.format, a, s);
}

template <bool WRITE>
static void launch(const CacheCall& c, hipStream_t s) {
    return c.slots64 ? launch<WRITE, int64_t>(c, s) : launch<WRITE, int32_t>(c, s);
}

}  // namespace hgsr

using namespace hgsr;

static int check_cache(const char* what, const CacheCall& c) {
    HGSR_REQUIRE(c.capacity >= 0 && c.capacity < (1ll << 31), "%s: capacity %lld outside [0, 2^31)", what,
                 (long long)c.capacity);
    HGSR_REQUIRE(c.n >= 0 && c.n < (1ll << 31) - 4096, "%s: %lld rows: too many", what, (long long)c.n);
    HGSR_REQUIRE(c.D >= 1 && c.D <= (1ll << 21), "%s: row length %lld outside [1, 2^21]", what, (long long)c.D);
    HGSR_REQUIRE(c.group == 16 || c.group == 32 || c.group == 64 || c.group == 128,
                 "%s: group of %d columns (16, 32, 64, 128)", what, c.group);
    HGSR_REQUIRE(c.format == HGSR_INT8 || c.format == HGSR_E4M3, "%s: unknown format", what);
    HGSR_REQUIRE(type_ok(c.type), "%s: unknown element type", what);
    HGSR_REQUIRE(c.cstride >= c.D && c.sstride >= (c.D + c.group - 1) / c.group && c.slots_stride >= 0 && c.xstride >= 0,
                 "%s: bad stride", what);
    HGSR_REQUIRE(c.slots || c.n <= c.capacity, "%s: %lld rows, %lld slots", what, (long long)c.n,
                 (long long)c.capacity);
    return HGSR_OK;
}

extern "C" size_t hgsr_rowcache_write_ws_bytes(int64_t capacity, int64_t n, int64_t D, int has_slots) {
    if (!has_slots || n <= 0 || capacity <= 0 || D < 1 || few_slots(n, D)) return 0;
    return align256(((size_t)(n + kSlotTile - 1) / kSlotTile + 1) * 4) + (size_t)capacity * sizeof(int32_t);
}

extern "C" int hgsr_rowcache_write(int64_t capacity, int64_t n, int64_t D, int group, int format, const void* x,
                                   int xtype, int64_t xstride, const void* slots, int slots64, int64_t slots_stride,
                                   void* codes, int64_t cstride, float* scales, int64_t sstride, void* ws,
                                   size_t ws_bytes, hgsr_stream_t stream) {
    const CacheCall c{capacity, n,      D,     cstride, sstride, slots_stride, xstride,
                      group,    format, xtype, slots64, slots,   codes,        const_cast<void*>(x), ws, scales};
    if (int st = check_cache("rowcache_write", c)) return st;
    if (n == 0 || capacity == 0) return HGSR_OK;
    HGSR_REQUIRE(x && codes && scales, "rowcache_write: null pointer");
    const size_t need = hgsr_rowcache_write_ws_bytes(capacity, n, D, slots != nullptr);
    if (need > ws_bytes || (need && !ws)) {
        set_error("rowcache_write: workspace of %zu bytes, %zu needed", ws ? ws_bytes : (size_t)0, need);
        return HGSR_EWORKSPACE;
    }
    hipStream_t s = as_stream(stream);
    {
        KernelTimer kt("rowcache_write", s);
        launch<true>(c, s);
    }
    return check_launch("rowcache_write");
}

extern "C" int hgsr_rowcache_read(int64_t capacity, int64_t n, int64_t D, int group, int format, const void* codes,
                                  int64_t cstride, const float* scales, int64_t sstride, const void* slots,
                                  int slots64, int64_t slots_stride, void* out, int otype, hgsr_stream_t stream) {
    const CacheCall c{capacity, n,      D,     cstride, sstride, slots_stride, D, group, format, otype, slots64, slots,
                      const_cast<void*>(codes), out, nullptr, const_cast<float*>(scales)};
    if (int st = check_cache("rowcache_read", c)) return st;
    if (n == 0) return HGSR_OK;
    HGSR_REQUIRE(out && (capacity == 0 || (codes && scales)), "rowcache_read: null pointer");
    hipStream_t s = as_stream(stream);
    {
        KernelTimer kt("rowcache_read", s);
        launch<false>(c, s);
    }
    return check_launch("rowcache_read");
}
