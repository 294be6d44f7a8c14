// Element types, vector accesses and index reads shared by the row-table kernels
// (embed.hip, rowcache.hip).
#pragma once
#include <type_traits>

#include "common.h"

namespace hgsr {

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

// VEC elements of T in registers (and, 16-byte aligned, in LDS)
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC > 16 ? 16 : sizeof(T) * VEC) Vec {
    T v[VEC];
};

// Moved from and to memory as accesses of up to 16 bytes wherever the elements lie: the hardware takes
// such accesses at any element's boundary.  So the columns that a lane holds, and with them the order
// of a sum, never depend on a tensor's address or row stride.
template <int BYTES>
struct Words;
template <>
struct Words<16> {
    typedef uint32_t reg __attribute__((ext_vector_type(4)));
    typedef reg word __attribute__((aligned(1), may_alias));
};
template <>
struct Words<8> {
    typedef uint32_t reg __attribute__((ext_vector_type(2)));
    typedef reg word __attribute__((aligned(1), may_alias));
};
template <>
struct Words<4> {
    typedef uint32_t reg;
    typedef reg word __attribute__((aligned(1), may_alias));
};
template <>
struct Words<2> {
    typedef uint16_t reg;
    typedef reg word __attribute__((aligned(1), may_alias));
};
template <typename T, int VEC>
struct Access {  // COUNT accesses of `word`
    static constexpr int BYTES = sizeof(T) * VEC < 16 ? sizeof(T) * VEC : 16, COUNT = sizeof(T) * VEC / BYTES;
    typedef typename Words<BYTES>::word word;
    typedef typename Words<BYTES>::reg reg;
};

template <typename T, int VEC>
__device__ __forceinline__ Vec<T, VEC> load_vec(const T* p) {
    typedef Access<T, VEC> A;
    Vec<T, VEC> x;
#pragma unroll
    for (int k = 0; k < A::COUNT; ++k) {
        const typename A::reg r = reinterpret_cast<const typename A::word*>(p)[k];
        __builtin_memcpy(reinterpret_cast<char*>(&x) + k * A::BYTES, &r, A::BYTES);
    }
    return x;
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, VEC>& x) {
    typedef Access<T, VEC> A;
#pragma unroll
    for (int k = 0; k < A::COUNT; ++k) {
        typename A::reg r;
        __builtin_memcpy(&r, reinterpret_cast<const char*>(&x) + k * A::BYTES, A::BYTES);
        reinterpret_cast<typename A::word*>(p)[k] = r;
    }
}
// the same, past the caches
template <typename T, int VEC>
__device__ __forceinline__ void stream_vec(T* p, const Vec<T, VEC>& x) {
    typedef Access<T, VEC> A;
#pragma unroll
    for (int k = 0; k < A::COUNT; ++k) {
        typename A::reg r;
        __builtin_memcpy(&r, reinterpret_cast<const char*>(&x) + k * A::BYTES, A::BYTES);
        __builtin_nontemporal_store(r, reinterpret_cast<typename A::word*>(p) + k);
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

// columns per lane: 8, 4, 2 or 1, at most `most` and no more than the row has
inline int vec_width(int most, int64_t dim) {
    int v = most;
    while (v > dim) v >>= 1;
    return v;
}

inline size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace hgsr
