// elements.h -- device helpers of the training operators: eight elements of a 16- or 32-bit type to and from fp32
// registers, and reductions over lanes, wavefronts and workgroups in a fixed order.
#ifndef SPANQR_ELEMENTS_H
#define SPANQR_ELEMENTS_H

#include <hip/hip_runtime.h>

#include <stdint.h>

namespace spanqr_dev {

typedef __bf16 bf16;
typedef _Float16 fp16;

// A row of odd length starts anywhere, so vectors are read and written at the element's own alignment: the memory
// pipeline takes 16-byte accesses at any address, and one form serves every row length and stride.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Pack8 {
    T v[8];
};

// elements [0, n) of p as fp32, n <= 8; the others 0
template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, float (&f)[8]) {
    if (n >= 8) {
        const Pack8<T> k = *reinterpret_cast<const Pack8<T>*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (float)k.v[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = i < n ? (float)p[i] : 0.0f;
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, int n, const float (&f)[8]) {
    if (n >= 8) {
        Pack8<T> k;
#pragma unroll
        for (int i = 0; i < 8; ++i) k.v[i] = (T)f[i];
        *reinterpret_cast<Pack8<T>*>(p) = k;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = (T)f[i];
    }
}

// Eight elements of a row of D >= 8 from `at` on, in two steps, so that many loads can be under way at once: fetch8 reads
// the last eight where fewer are left (no branch, nothing past the row), and settle8 moves those to their place and
// puts 0 behind them. n: how many are left, 0 to 8.
template <typename T>
__device__ __forceinline__ Pack8<T> fetch8(const T* row, long D, long at) {
    return *reinterpret_cast<const Pack8<T>*>(row + (at < D - 8 ? at : D - 8));
}
template <typename T>
__device__ __forceinline__ void settle8(const Pack8<T>& k, int n, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)k.v[i];
    if (n < 8) {
#pragma unroll
        for (int b = 4; b > 0; b >>= 1) {   // by 8 - n places
            const bool move = (8 - n) & b;
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = move ? (i + b < 8 ? f[i + b] : 0.0f) : f[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = i < n ? f[i] : 0.0f;
    }
}

// makes the compiler unpack k again behind this point instead of keeping what it unpacked before
template <typename T>
__device__ __forceinline__ void again(Pack8<T>& k) {
    constexpr int N = sizeof(T) * 8 / 4;
    struct Words { uint32_t w[N]; };
    Words b = __builtin_bit_cast(Words, k);
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(b.w[i]));
    k = __builtin_bit_cast(Pack8<T>, b);
}

// the larger of two magnitudes; NaN if either is
__device__ __forceinline__ float nan_max(float a, float b) { return (b > a || b != b) ? b : a; }

struct Sum {
    template <typename A>
    __device__ __forceinline__ static A of(A a, A b) { return a + b; }
};
struct NanMax {
    __device__ __forceinline__ static float of(float a, float b) { return nan_max(a, b); }
};

// over LANES neighbouring lanes (a power of two up to 64); every lane gets the same value
template <int LANES, typename OP, typename A>
__device__ __forceinline__ A reduce_lanes(A v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = OP::of(v, __shfl_xor(v, o));
    return v;
}

// over THREADS threads (a multiple of 64) that share `slot` (THREADS / 64 values in LDS). Two barriers: the slot can be
// used again at once.
template <int THREADS, typename OP, typename A>
__device__ __forceinline__ A reduce_threads(A v, A* slot) {
    v = reduce_lanes<64, OP>(v);
    if (THREADS > 64) {
        const int w = (threadIdx.x % THREADS) >> 6;
        if ((threadIdx.x & 63) == 0) slot[w] = v;
        __syncthreads();
        v = slot[0];
#pragma unroll
        for (int i = 1; i < THREADS / 64; ++i) v = OP::of(v, slot[i]);
        __syncthreads();
    }
    return v;
}

}  // namespace spanqr_dev

#endif  // SPANQR_ELEMENTS_H
