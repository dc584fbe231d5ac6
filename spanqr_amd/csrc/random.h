// random.h -- the numbers that dropout goes by, from a counter: nothing is kept but a seed, and the backward pass makes the
// same ones again.
//
// Philox-4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011): four words of
// 32 bits from a counter of four and a key of two. Each word gives two numbers of 16 bits, so one counter serves eight
// neighbouring elements of a row: (piece, row mod 2^32, row / 2^32, index), the seed's words being the key. An element's number
// depends on its row and column alone, not on strides, types or the way a kernel divides its work. 16 bits make the
// probability a multiple of 2^-16, and the factor is that of the multiple; 32 bits an element would make dropout of
// 16-bit types wait for the multiplier instead of the memory.
#ifndef SPANQR_RANDOM_H
#define SPANQR_RANDOM_H

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

namespace spanqr_dev {

struct Dropout {
    uint32_t below;            // numbers below this are dropped; 0: nothing is, and no numbers are made
    float factor;              // of the others: 65536 / (65536 - below)
    uint64_t seed;
    const uint64_t* seed_at;   // on the device, read instead where it is not null
    uint32_t index;

    // the seed, in scalar registers (the rounds' keys too, then)
    __device__ __forceinline__ uint64_t key() const {
        const uint64_t k = below != 0 && seed_at != nullptr ? *seed_at : seed;
        return (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(k >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)k);
    }

    // elements 8 piece to 8 piece + 7 of a row: 0 where dropped (also what is infinite or NaN), the others times the factor
    __device__ __forceinline__ void thin(uint64_t key, long row, long piece, float (&v)[8]) const {
        if (below == 0) return;
        uint32_t c0 = (uint32_t)piece, c1 = (uint32_t)row, c2 = (uint32_t)((uint64_t)row >> 32), c3 = index;
        uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
        for (int r = 0; r < 10; ++r) {
            const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
            c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
            c1 = (uint32_t)b;
            c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
            c3 = (uint32_t)a;
            k0 += 0x9E3779B9u;
            k1 += 0xBB67AE85u;
        }
        const uint32_t word[4] = {c0, c1, c2, c3};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t number = i & 1 ? word[i >> 1] >> 16 : word[i >> 1] & 0xFFFFu;
            v[i] = number < below ? 0.0f : v[i] * factor;
        }
    }
};

// p in 16 bits, to nearest even; -1 where it leaves nothing or is no probability
inline int dropped_below(double p) {
    if (!(p >= 0.0 && p < 1.0)) return -1;
    const double n = rint(65536.0 * p);
    return n < 65536.0 ? (int)n : -1;
}

}  // namespace spanqr_dev

#endif  // SPANQR_RANDOM_H
