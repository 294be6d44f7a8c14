// Element types, vector accesses and index reads shared by the row-table kernels
// (embed.hip, rowcache.hip).
#pragma once
#include <type_traits>

#include "common.h"

namespace hgsr {

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

// VEC elements of T in registers, moved as one access of up to 16 bytes (two for 8 floats)
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC > 16 ? 16 : sizeof(T) * VEC) Vec {
    T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ Vec<T, VEC> load_vec(const T* p) {
    return *reinterpret_cast<const Vec<T, VEC>*>(p);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, VEC>& x) {
    *reinterpret_cast<Vec<T, VEC>*>(p) = x;
}

// the same, past the caches
template <typename T, int VEC>
__device__ __forceinline__ void stream_vec(T* p, const Vec<T, VEC>& x) {
    if constexpr (sizeof(x) % 4 == 0) {
        constexpr int W = sizeof(x) / 4 < 4 ? sizeof(x) / 4 : 4;
        typedef uint32_t words __attribute__((ext_vector_type(W)));
#pragma unroll
        for (int k = 0; k < (int)sizeof(x) / (4 * W); ++k)
            __builtin_nontemporal_store(reinterpret_cast<const words*>(&x)[k], reinterpret_cast<words*>(p) + k);
    } else {
        store_vec<T, VEC>(p, x);
    }
}
// Rows of more bytes than the L2 caches hold (8 x 4 MB) are stored past them: what reads them next
// finds none there anyway, and the lookup of 500k rows of 32 floats takes 21.2 us instead of 23.9, of
// 16k rows of 2048 bf16 16.2 instead of 18.4.
inline int stream_out(int64_t bytes) { return bytes > (32 << 20); }

// Row numbers, I = int32_t or int64_t, `stride` elements apart (0: one number for every entry).
// Anything outside [0, limit) comes back as `limit`, the number of no row.  The type is a template
// argument: a branch on it around each load keeps a lane's loads from being in flight together
// (the count of 500k ids took 15 us instead of 9).
template <typename I>
struct RowIds {
    const I* p;
    int64_t stride;
    __device__ __forceinline__ uint32_t get(int64_t i, uint32_t limit) const {
        const typename std::make_unsigned<I>::type v = p[i * stride];
        return v < limit ? (uint32_t)v : limit;
    }
};

// i / d for i < 2^31 by one 32x32 product: with p = 31 + ceil(log2 d) and m = ceil(2^p / d) < 2^32,
// m d - 2^p < 2^(p - 31), so i m / 2^p exceeds i / d by less than 1 / d and the floors agree.
struct FastDiv {
    uint32_t d, m, p;
    __device__ __forceinline__ uint32_t div(uint32_t i) const { return (uint32_t)(((uint64_t)i * m) >> p); }
};
inline FastDiv fast_div(uint32_t d) {
    uint32_t l = 0;
    while ((1ull << l) < d) ++l;
    const uint32_t p = 31 + l;
    return {d, (uint32_t)(((1ull << p) + d - 1) / d), p};
}

inline int elem_size(int type) { return type == HGSR_F32 ? 4 : 2; }
inline bool type_ok(int type) { return type == HGSR_F32 || type == HGSR_F16 || type == HGSR_BF16; }

// The largest of 1, 2, 4, 8 elements (at most `most`) that divides the row length and the row
// stride and at which rows of `size`-byte elements start on an access boundary
inline int vec_width(int most, int64_t dim, int64_t stride, const void* base, int size) {
    int v = most;
    while (v > 1) {
        const int bytes = v * size > 16 ? 16 : v * size;
        if (dim % v == 0 && stride % v == 0 && (uintptr_t)base % bytes == 0) break;
        v >>= 1;
    }
    return v;
}

inline size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace hgsr
