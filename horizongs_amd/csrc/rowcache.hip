// K19: a cache of rows held in 8 bits -- quantised as they are written into their slots, and read
// back by slot (the anchor features of a merged scene, or any rows kept for later reads).
//
//   write  s = max(max |x| over a group of columns * (1 / top), 2^-100),  code = round(x / s)
//   read   x' = code * s
//
// Both are bound by memory: a lane moves 4 (f32) or 8 (16-bit) consecutive columns of a row, the
// lanes of a group find its maximum among themselves.
#include "rows.h"

namespace hgsr {

constexpr float kScaleFloor = 0x1p-100f;

struct CacheArgs {
    uint32_t capacity, chunks, width;  // chunks: lanes' pieces of this launch; width: pieces per row
    FastDiv per_row;
    int64_t row0, D;
    int group, glog;                   // group = 1 << glog columns
    uint8_t* codes;
    float* scales;
    int64_t cstride, sstride;
    RowIds slots;                      // slots.p == nullptr: slot i
    void* x;                           // rows written, or the rows that a read fills
    int64_t xstride;
    const int32_t* last;               // write: the last row of each named slot (nullable)
};

__device__ __forceinline__ uint32_t slot_of(const CacheArgs& a, int64_t i) {
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

template <int FMT>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    if (FMT == HGSR_INT8)
        return ((uint32_t)(int)rintf(a) & 255u) | ((uint32_t)(int)rintf(b) & 255u) << 8 |
               ((uint32_t)(int)rintf(c) & 255u) << 16 | (uint32_t)(int)rintf(d) << 24;
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
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

// the last row that names each slot: cleared where it will be read, then the largest row number
__global__ __launch_bounds__(256) void slot_clear_kernel(uint32_t n, RowIds slots, uint32_t capacity,
                                                         int32_t* __restrict__ last) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const uint32_t c = slots.get(i, capacity);
    if (c < capacity) last[c] = -1;
}
__global__ __launch_bounds__(256) void slot_last_kernel(uint32_t n, RowIds slots, uint32_t capacity,
                                                        int32_t* __restrict__ last) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const uint32_t c = slots.get(i, capacity);
    if (c < capacity) atomicMax(&last[c], (int32_t)i);
}

// VEC consecutive columns per lane; ALIGNED: whole pieces, moved as vectors
template <typename XT, int FMT, int VEC, bool ALIGNED>
__global__ __launch_bounds__(256) void rowcache_write_kernel(const CacheArgs a) {
    const uint32_t c = blockIdx.x * 256 + threadIdx.x;
    const uint32_t r = a.per_row.div(c < a.chunks ? c : 0);
    const int64_t row = a.row0 + r, col = (int64_t)(c - r * a.per_row.d) * VEC;
    uint32_t slot = c < a.chunks ? slot_of(a, row) : a.capacity;
    if (slot < a.capacity && a.last && a.last[slot] != (int32_t)row) slot = a.capacity;
    const bool on = slot < a.capacity && col < a.D;
    float x[VEC] = {};
    if (on) {
        const XT* p = static_cast<const XT*>(a.x) + row * a.xstride + col;
        if (ALIGNED) {
            const Vec<XT, VEC> v = load_vec<XT, VEC>(p);
#pragma unroll
            for (int k = 0; k < VEC; ++k) x[k] = (float)v.v[k];
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                if (col + k < a.D) x[k] = (float)p[k];
        }
    }
    // the largest magnitude of the group as bits: infinities and NaN lie above every number
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < VEC; ++k) m = max(m, __float_as_uint(x[k]) & 0x7fffffffu);
    const int lanes = a.group / VEC;  // a power of two, <= 32
    for (int d = 1; d < lanes; d <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
    if (!on) return;
    const bool finite = m < 0x7f800000u;
    const float per = FMT == HGSR_INT8 ? 1.0f / 127.0f : 1.0f / 448.0f;
    const float s = fmaxf(__uint_as_float(m) * per, kScaleFloor), inv = 1.0f / s;
    uint32_t w[VEC / 4];
#pragma unroll
    for (int k = 0; k < VEC; k += 4) {
        float q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = finite ? quotient_odd(x[k + j], s, inv) : 0.0f;
        w[k / 4] = encode4<FMT>(q[0], q[1], q[2], q[3]);
    }
    uint8_t* to = a.codes + (int64_t)slot * a.cstride + col;
    if (ALIGNED) {
        Vec<uint32_t, VEC / 4> o;
#pragma unroll
        for (int k = 0; k < VEC / 4; ++k) o.v[k] = w[k];
        store_vec<uint32_t, VEC / 4>(reinterpret_cast<uint32_t*>(to), o);
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            if (col + k < a.D) to[k] = (uint8_t)(w[k / 4] >> (8 * (k & 3)));
    }
    if ((col & (a.group - 1)) == 0)
        a.scales[(int64_t)slot * a.sstride + (col >> a.glog)] = finite ? s : __builtin_nanf("");
}

// -------------------------------------------------------------------------------------- read

template <typename OT, int FMT, int VEC, bool ALIGNED>
__global__ __launch_bounds__(256) void rowcache_read_kernel(const CacheArgs a) {
    const uint32_t c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.chunks) return;
    const uint32_t r = a.per_row.div(c);
    const int64_t row = a.row0 + r, col = (int64_t)(c - r * a.per_row.d) * VEC;
    const uint32_t slot = slot_of(a, row);
    float x[VEC] = {};
    if (slot < a.capacity) {
        const uint8_t* p = a.codes + (int64_t)slot * a.cstride + col;
        const float s = a.scales[(int64_t)slot * a.sstride + (col >> a.glog)];
        uint32_t w[VEC / 4];
        if (ALIGNED) {
            const Vec<uint32_t, VEC / 4> v = load_vec<uint32_t, VEC / 4>(reinterpret_cast<const uint32_t*>(p));
#pragma unroll
            for (int k = 0; k < VEC / 4; ++k) w[k] = v.v[k];
        } else {
#pragma unroll
            for (int k = 0; k < VEC / 4; ++k) w[k] = 0;
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                if (col + k < a.D) w[k / 4] |= (uint32_t)p[k] << (8 * (k & 3));
        }
#pragma unroll
        for (int k = 0; k < VEC; k += 4) decode4<FMT>(w[k / 4], x + k);
#pragma unroll
        for (int k = 0; k < VEC; ++k) x[k] *= s;
    }
    OT* to = static_cast<OT*>(a.x) + row * a.D + col;
    if (ALIGNED) {
        Vec<OT, VEC> o;
#pragma unroll
        for (int k = 0; k < VEC; ++k) o.v[k] = (OT)x[k];
        store_vec<OT, VEC>(to, o);
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            if (col + k < a.D) to[k] = (OT)x[k];
    }
}

// ---------------------------------------------------------------------------------- launches

template <typename T, int FMT, int VEC>
static void launch(bool write, bool aligned, const CacheArgs& a, hipStream_t s) {
    const dim3 grid((a.chunks + 255) / 256), block(256);
    if (write && aligned)
        hipLaunchKernelGGL((rowcache_write_kernel<T, FMT, VEC, true>), grid, block, 0, s, a);
    else if (write)
        hipLaunchKernelGGL((rowcache_write_kernel<T, FMT, VEC, false>), grid, block, 0, s, a);
    else if (aligned)
        hipLaunchKernelGGL((rowcache_read_kernel<T, FMT, VEC, true>), grid, block, 0, s, a);
    else
        hipLaunchKernelGGL((rowcache_read_kernel<T, FMT, VEC, false>), grid, block, 0, s, a);
}

template <typename T, int VEC>
static void launch(bool write, int format, int64_t n, CacheArgs a, hipStream_t s) {
    bool aligned = a.D % VEC == 0 && a.cstride % VEC == 0 && (uintptr_t)a.codes % VEC == 0;
    aligned = aligned && (uintptr_t)a.x % 16 == 0 && a.xstride % VEC == 0;
    // a write's rows are whole groups of lanes, so that no group crosses a wave
    const int64_t per_row = write ? (a.D + a.group - 1) / a.group * (a.group / VEC) : (a.D + VEC - 1) / VEC;
    const int64_t most = ((int64_t)1 << 30) / per_row;
    a.per_row = fast_div((uint32_t)per_row);
    for (a.row0 = 0; a.row0 < n; a.row0 += most) {
        a.chunks = (uint32_t)((n - a.row0 < most ? n - a.row0 : most) * per_row);
        if (format == HGSR_INT8)
            launch<T, HGSR_INT8, VEC>(write, aligned, a, s);
        else
            launch<T, HGSR_E4M3, VEC>(write, aligned, a, s);
    }
}

static void launch(bool write, int type, int format, int64_t n, const CacheArgs& a, hipStream_t s) {
    if (type == HGSR_F32)
        launch<float, 4>(write, format, n, a, s);
    else if (type == HGSR_F16)
        launch<f16_t, 8>(write, format, n, a, s);
    else
        launch<bf16_t, 8>(write, format, n, a, s);
}

}  // namespace hgsr

using namespace hgsr;

static int cache_args(const char* what, int64_t capacity, int64_t n, int64_t D, int group, int format, int type,
                      int64_t cstride, int64_t sstride, const void* slots, int slots64, int64_t slots_stride,
                      CacheArgs& a) {
    HGSR_REQUIRE(capacity >= 0 && capacity < (1ll << 31), "%s: capacity %lld outside [0, 2^31)", what,
                 (long long)capacity);
    HGSR_REQUIRE(n >= 0 && n < (1ll << 31) - 256, "%s: %lld rows: too many", what, (long long)n);
    HGSR_REQUIRE(D >= 1 && D <= (1ll << 21), "%s: row length %lld outside [1, 2^21]", what, (long long)D);
    HGSR_REQUIRE(group == 16 || group == 32 || group == 64 || group == 128, "%s: group of %d columns (16, 32, 64, 128)",
                 what, group);
    HGSR_REQUIRE(format == HGSR_INT8 || format == HGSR_E4M3, "%s: unknown format", what);
    HGSR_REQUIRE(type_ok(type), "%s: unknown element type", what);
    HGSR_REQUIRE(cstride >= D && sstride >= (D + group - 1) / group && slots_stride >= 0, "%s: bad stride", what);
    HGSR_REQUIRE(slots || n <= capacity, "%s: %lld rows, %lld slots", what, (long long)n, (long long)capacity);
    a.capacity = (uint32_t)capacity;
    a.D = D;
    a.group = group;
    a.glog = group == 16 ? 4 : group == 32 ? 5 : group == 64 ? 6 : 7;
    a.cstride = cstride;
    a.sstride = sstride;
    a.slots = RowIds{slots, slots_stride, slots64};
    return HGSR_OK;
}

extern "C" size_t hgsr_rowcache_write_ws_bytes(int64_t capacity, int64_t n, int has_slots) {
    return has_slots && n > 1 && capacity > 0 ? (size_t)capacity * sizeof(int32_t) : 0;
}

extern "C" int hgsr_rowcache_write(int64_t capacity, int64_t n, int64_t D, int group, int format, const void* x,
                                   int xtype, int64_t xstride, const void* slots, int slots64, int64_t slots_stride,
                                   void* codes, int64_t cstride, float* scales, int64_t sstride, void* ws,
                                   size_t ws_bytes, hgsr_stream_t stream) {
    CacheArgs a{};
    if (int st = cache_args("rowcache_write", capacity, n, D, group, format, xtype, cstride, sstride, slots, slots64,
                            slots_stride, a))
        return st;
    HGSR_REQUIRE(xstride >= 0, "rowcache_write: negative stride");
    if (n == 0 || capacity == 0) return HGSR_OK;
    HGSR_REQUIRE(x && codes && scales, "rowcache_write: null pointer");
    a.x = const_cast<void*>(x);
    a.xstride = xstride;
    a.codes = static_cast<uint8_t*>(codes);
    a.scales = scales;
    hipStream_t s = as_stream(stream);
    KernelTimer kt("rowcache_write", s);
    if (slots && n > 1) {
        const size_t need = hgsr_rowcache_write_ws_bytes(capacity, n, 1);
        if (!ws || ws_bytes < need) {
            set_error("rowcache_write: workspace of %zu bytes, %zu needed", ws_bytes, need);
            return HGSR_EWORKSPACE;
        }
        int32_t* last = static_cast<int32_t*>(ws);
        const dim3 grid((unsigned)((n + 255) / 256));
        hipLaunchKernelGGL(slot_clear_kernel, grid, dim3(256), 0, s, (uint32_t)n, a.slots, a.capacity, last);
        hipLaunchKernelGGL(slot_last_kernel, grid, dim3(256), 0, s, (uint32_t)n, a.slots, a.capacity, last);
        a.last = last;
    }
    launch(true, xtype, format, n, a, s);
    return check_launch("rowcache_write");
}

extern "C" int hgsr_rowcache_read(int64_t capacity, int64_t n, int64_t D, int group, int format, const void* codes,
                                  int64_t cstride, const float* scales, int64_t sstride, const void* slots,
                                  int slots64, int64_t slots_stride, void* out, int otype, hgsr_stream_t stream) {
    CacheArgs a{};
    if (int st = cache_args("rowcache_read", capacity, n, D, group, format, otype, cstride, sstride, slots, slots64,
                            slots_stride, a))
        return st;
    if (n == 0) return HGSR_OK;
    HGSR_REQUIRE(out && (capacity == 0 || (codes && scales)), "rowcache_read: null pointer");
    a.x = out;
    a.xstride = D;
    a.codes = const_cast<uint8_t*>(static_cast<const uint8_t*>(codes));
    a.scales = const_cast<float*>(scales);
    hipStream_t s = as_stream(stream);
    KernelTimer kt("rowcache_read", s);
    launch(false, otype, format, n, a, s);
    return check_launch("rowcache_read");
}
