// rows.h -- what the kernels share that work on rows of any length with the row in registers (norm.hip, block.hip): which
// threads have a row, its pieces of eight elements, weights, and how many workgroups there are.
#ifndef SPANQR_ROWS_H
#define SPANQR_ROWS_H

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

// piece `at` of a row; WHOLE: the row has 8 elements at least (shorter ones are read one by one)
template <bool WHOLE, typename T>
__device__ __forceinline__ Pack8<T> piece(const T* row, long D, long at, int n) {
    if constexpr (WHOLE) return fetch8(row, D, at);
    Pack8<T> k;
#pragma unroll
    for (int i = 0; i < 8; ++i) k.v[i] = i < n ? row[at + i] : (T)0.0f;
    return k;
}
template <bool WHOLE, typename T>
__device__ __forceinline__ void settle(const Pack8<T>& k, int n, float (&f)[8]) {
    if constexpr (WHOLE) {
        settle8(k, n, f);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (float)k.v[i];
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
