// rows.h -- what the kernels share that work on rows of any length with the row in registers (norm.hip, block.hip): which
// threads have a row, its pieces of eight elements, weights, and how many workgroups there are.
#ifndef SPANQR_ROWS_H
#define SPANQR_ROWS_H

#include <type_traits>

#include "elements.h"

#include "../../include/spanqr.h"

namespace spanqr_dev {

// eight weights as fp32; 1 without weights
__device__ __forceinline__ void load_weight(const void* w, int type, long at, int n, float (&f)[8]) {
    if (w == nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = 1.0f;
    } else if (type == SPANQR_BF16) {
        load8((const bf16*)w + at, n, f);
    } else if (type == SPANQR_FP16) {
        load8((const fp16*)w + at, n, f);
    } else {
        load8((const float*)w + at, n, f);
    }
}

// elements of the piece at `at` that are inside the row (0 to 8)
__device__ __forceinline__ int inside(long D, long at) { return D - at >= 8 ? 8 : D > at ? (int)(D - at) : 0; }

// the sum over LANES (16 or 64) neighbouring lanes, in every one of them, without going through LDS
template <int LANES>
__device__ __forceinline__ float sum_lanes(float v) {
    const auto lane = [](float x, auto ctrl) {
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xF, 0xF, true));
    };
    v += lane(v, std::integral_constant<int, 0xB1>{});    // the neighbour's of two
    v += lane(v, std::integral_constant<int, 0x4E>{});    // the other two's of four
    v += lane(v, std::integral_constant<int, 0x141>{});   // the other four's of eight
    v += lane(v, std::integral_constant<int, 0x140>{});   // the other eight's of sixteen
    if constexpr (LANES == 64) {
        const auto both = [](auto r) {
            const uint32_t a = r[0], b = r[1];   // (a bit_cast of a vector's element takes the first one)
            return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
        };
        uint32_t u = __builtin_bit_cast(uint32_t, v);
        u = __builtin_bit_cast(uint32_t, both(__builtin_amdgcn_permlane16_swap(u, u, false, false)));
        v = both(__builtin_amdgcn_permlane32_swap(u, u, false, false));
    }
    return v;
}

// Threads of a row: GROUP lanes of a wavefront (16 or 64; then a workgroup of 256 threads has several rows), or with GROUP
// 0 the whole workgroup, of any number of wavefronts.
template <int GROUP>
struct Group {
    static constexpr int MOST = GROUP ? 256 : 1024;
    __device__ __forceinline__ static int size() { return GROUP ? GROUP : (int)blockDim.x; }
    __device__ __forceinline__ static int rows() { return GROUP ? 256 / GROUP : 1; }
    __device__ __forceinline__ static int lane() { return GROUP ? threadIdx.x % GROUP : threadIdx.x; }
    __device__ __forceinline__ static int index() { return GROUP ? threadIdx.x / GROUP : 0; }
    // N values over the group's threads. One barrier: `slot` ([N][16]) may be used again only behind another one.
    template <typename OP, int N>
    __device__ __forceinline__ static void reduce(float (&v)[N], float (*slot)[16]) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = reduce_lanes<GROUP ? GROUP : 64, OP>(v[i]);
        across<OP>(v, slot);
    }
    // sums, in another order
    template <int N>
    __device__ __forceinline__ static void sum(float (&v)[N], float (*slot)[16]) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = sum_lanes<GROUP ? GROUP : 64>(v[i]);
        across<Sum>(v, slot);
    }

private:
    template <typename OP, int N>
    __device__ __forceinline__ static void across(float (&v)[N], float (*slot)[16]) {
        if constexpr (GROUP == 0) {
            const int waves = blockDim.x >> 6;
            if ((threadIdx.x & 63) == 0) {
#pragma unroll
                for (int i = 0; i < N; ++i) slot[i][threadIdx.x >> 6] = v[i];
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = slot[i][0];
            for (int w = 1; w < waves; ++w) {
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] = OP::of(v[i], slot[i][w]);
            }
        }
    }
};

// Piece `at` of a row. WHOLE 1: the row has 8 elements at least (shorter ones, 0, are read one by one); 2: its length is a
// multiple of 8, so that a piece is all there or not at all.
template <int WHOLE, typename T>
__device__ __forceinline__ Pack8<T> piece(const T* row, long D, long at, int n) {
    if constexpr (WHOLE != 0) return fetch8(row, D, at);
    Pack8<T> k;
#pragma unroll
    for (int i = 0; i < 8; ++i) k.v[i] = i < n ? row[at + i] : (T)0.0f;
    return k;
}
template <int WHOLE, typename T>
__device__ __forceinline__ void settle(const Pack8<T>& k, int n, float (&f)[8]) {
    if constexpr (WHOLE == 1) {
        settle8(k, n, f);
    } else if constexpr (WHOLE == 2) {
        struct Words { uint32_t w[2 * sizeof(T)]; } b = __builtin_bit_cast(Words, k);
        const uint32_t mask = n ? 0xFFFFFFFFu : 0u;
#pragma unroll
        for (int i = 0; i < 2 * (int)sizeof(T); ++i) b.w[i] &= mask;
        const Pack8<T> m = __builtin_bit_cast(Pack8<T>, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (float)m.v[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = i < n ? (float)k.v[i] : 0.0f;
    }
}

// Threads of a row and pieces a thread.
struct Split {
    int group, nch;   // group 16 or 64: lanes of a wavefront; else (64 and `block`) a workgroup
    bool block;
};

// workgroups for `rows` rows, each of about as many rows as the others, `most` at most
inline int grid_of(long rows, const Split& s, int most) {
    const int per = s.block ? 1 : 256 / s.group;
    const long need = (rows + per - 1) / per, turns = (need + most - 1) / most;
    return turns < 1 ? 0 : (int)((need + turns - 1) / turns);
}

}  // namespace spanqr_dev

#endif  // SPANQR_ROWS_H
