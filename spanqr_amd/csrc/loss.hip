// loss.hip -- softmax cross entropy over a large vocabulary from the hidden states and the head's weights, without
// keeping the logits, and its gradients.
//
//   z = x W^T [N, V],  lse_i = log sum_j exp z_ij,  loss_i = w_i (lse_i - z_i,t_i)      (w_i = 0 where t_i is ignored)
//   G_ij = w_i (exp(z_ij - lse_i) - [j = t_i]),  dx = a G W,  dW = a G^T x      (a = 1, or 1 / tokens that count)
//
// Three products of 2 N H V operations each. The product of the logits ends in its own softmax statistics: for
// 64 or 128 neighbouring columns of a token it leaves the maximum m and the sum of exp(z - m), and, where gradients are wanted,
// the exponentials p = exp(z - m) themselves, rounded to the 16-bit type once. One pass over p turns them into G
// (times exp(m - lse), the target's element from its fp32 logit), and G goes into the other two products. So nothing
// is multiplied twice, and what is held is 16 bits an element for as many tokens at a time as the workspace takes.
#include <type_traits>

#include "elements.h"
#include "host.h"

using namespace spanqr_dev;
using spanqr_host::error;
using spanqr_host::launched;

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 fp16x8 __attribute__((ext_vector_type(8)));

constexpr float LOG2E = 1.44269504088896340736f;

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }

template <typename T>
struct Vec;
template <>
struct Vec<bf16> {
    typedef bf16x8 x8;
    __device__ __forceinline__ static f32x4 mfma(x8 a, x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Vec<fp16> {
    typedef fp16x8 x8;
    __device__ __forceinline__ static f32x4 mfma(x8 a, x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};

// G is held in 16 bits; half precision has it times 2^10, so that probabilities down to 2^-34 stay normal or at least
// count (bf16 has fp32's exponents)
template <typename T>
constexpr float g_scale() { return sizeof(T) == 2 && std::is_same<T, fp16>::value ? 1024.0f : 1.0f; }

// C[n][m] = sum over k of A(m, k) B(n, k), for the three products:
//   logits  m = vocabulary (A = W rows),    n = token (B = x rows),         k = hidden
//   dx      m = hidden     (A = W columns), n = token (B = G rows),         k = vocabulary
//   dW      m = hidden     (A = x columns), n = vocabulary (B = G columns), k = token
// With m along the matrix instruction's rows a lane holds neighbouring elements of one row of C.
struct ProductArgs {
    long M, N, K;
    const void *A, *B;
    long lda, ldb;               // elements between rows as they lie in memory, multiples of 8, below 2^22
    const void* zeros;           // 16 bytes of zeros: what is read past K
    int m_tiles, n_tiles, splits;
    long split_k;                // the k of one split, a multiple of 64
    // logits
    const long* target;          // of token 0 of this piece
    float* zt;                   // the target's logit
    float2* stat;                // [token][segs]: maximum, sum
    long segs;
    void* p;                     // exponentials [token][ldp], or null
    long ldp;
    // dx, dW
    void* C;
    long ldc;
    int vector;                  // C takes 8-byte stores
    float* acc;                  // fp32 sums [split][N][ldacc], or null: C directly
    long ldacc;
    int add;                     // add to what acc holds
    const float* alpha;
};

enum { LOGITS, OUT };

typedef __attribute__((address_space(3))) char lds_char;
typedef short s16x4 __attribute__((ext_vector_type(4)));

// 16 bytes a lane from base + off to LDS at `lds` + 16 lane, asynchronously (counted by vmcnt). In inline asm because the
// compiler would wait for it before any later LDS read; it has no register output.
__device__ __forceinline__ void load_lds(const void* base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory");
}
__device__ __forceinline__ void load_lds_any(const void* at, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(at) : "memory");
}

constexpr int BK = 32, STAGES = 4;   // k of a step, and steps in LDS

// One operand's tiles of R rows (m or n) by 32 k in LDS, and the way there and into registers.
// ROWS (k neighbours in memory): R rows of 64 bytes; the 16-byte chunk c of a row lies at c ^ swizzle(row), so that
// the 16 rows a matrix instruction reads spread over the banks (a 16-byte read takes lanes 0-3, 12-15, 20-27 of each 32
// together, and then the others: 4 clocks this way, 8 with row / 4 itself in the place of its negative).
// Otherwise (m or n neighbours): 32 k-rows of 2 R bytes, read by the transposing LDS read (16 lanes fetch 4 k-rows of
// 16 columns and each gets one column's 4 k); the 32-byte block b of a row lies at b ^ swizzle(k).
// SPREAD (ROWS, logits): row r of subtile i of a group of 64 is row 16 (r / 4) + 4 i + r % 4, so that a lane's results
// of four subtiles are 16 neighbouring columns of C.
template <typename T, bool ROWS, bool SPREAD, int R, int WAVES, int SUB>
struct Tile {
    typedef typename Vec<T>::x8 x8;
    static constexpr int BYTES = R * 2 * BK;
    static constexpr int LOADS = BYTES / 1024 / WAVES;   // instructions of 64 x 16 bytes per wavefront and step
    static constexpr int RB = 2 * R, PER = 1024 / RB, LPR = RB / 16;

    const char* base;            // of this tile's rows at k = 0
    long step;                   // bytes for 32 k
    uint32_t off[LOADS];
    uint32_t dst;                // LDS of the wavefront's first instruction
    uint32_t at[ROWS ? 1 : SUB]; // LDS of the lane's fragments

    __device__ __forceinline__ static int swizzle(int i) {   // of a row, or of a k
        if constexpr (ROWS)
            return -(SPREAD ? i >> 4 : i >> 2) & 3;
        else
            return R >= 256 ? (i & 3) | (i >> 3 & 3) << 2 : R == 128 ? (i & 3) | (i >> 3 & 1) << 2 : (i >> 1 & 1) | (i >> 3 & 1) << 1;
    }

    __device__ __forceinline__ void init(const void* src, long ld, long rows, long r0, long k0, lds_char* lds, int wave, int lane,
                                         int first) {
        const int lo = lane & 15, hi = lane >> 4;
        const uint32_t lds0 = (uint32_t)(uintptr_t)lds;
        dst = __builtin_amdgcn_readfirstlane(lds0 + wave * LOADS * 1024);
        if constexpr (ROWS) {
            base = (const char*)src + 2 * (r0 * ld + k0);
            step = 2 * BK;
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int row = 16 * (wave * LOADS + i) + (lane >> 2);
                const long r = r0 + row < rows ? row : rows - 1 - r0;   // rows past the end: any, not used
                off[i] = (uint32_t)(2 * r * ld + 16 * ((lane & 3) ^ swizzle(row)));
            }
            const int row = SPREAD ? 16 * (lo >> 2) + (lo & 3) : lo;
            at[0] = lds0 + (first + row) * 64 + 16 * (hi ^ swizzle(row));
        } else {
            base = (const char*)src + 2 * (r0 + k0 * ld);
            step = 2 * BK * ld;
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int k = (wave * LOADS + i) * PER + lane / LPR, c = lane % LPR;
                int col = 16 * ((c >> 1) ^ swizzle(k)) + 8 * (c & 1);
                if (r0 + col >= rows) col = 0;
                off[i] = (uint32_t)(2 * (k * ld + col));
            }
            const int k = 8 * hi + (lo >> 2);
#pragma unroll
            for (int i = 0; i < SUB; ++i)
                at[i] = lds0 + k * RB + (((first / 16 + i) ^ swizzle(k)) << 5) + 8 * (lo & 3);
        }
    }

    // Stages 0 and 1 are those of this turn of the loop, 2 and 3 of the other. The bit is clear in every fragment's and
    // every load's address: an operand's stages start on a multiple of all of them.
    __device__ __forceinline__ void turn() {
        dst ^= 2 * BYTES;
#pragma unroll
        for (int i = 0; i < (ROWS ? 1 : SUB); ++i) at[i] ^= 2 * BYTES;
    }

    // instruction i of the load of k 32 t on into stage `stage`
    __device__ __forceinline__ void load(int t, int stage, int i) const {
        load_lds(base + t * step, off[i], (dst ^ (stage & 2) * BYTES) + (stage & 1) * BYTES + i * 1024);
    }
    // the whole of it where only `left` k are left (none where left <= 0)
    __device__ __forceinline__ void load_end(int t, int stage, int left, const void* zeros, int wave, int lane) const {
        const char* b = base + t * step;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            int k;
            if constexpr (ROWS)
                k = 8 * ((lane & 3) ^ swizzle(16 * (wave * LOADS + i) + (lane >> 2)));
            else
                k = (wave * LOADS + i) * PER + lane / LPR;
            load_lds_any(k < left ? (const void*)(b + off[i]) : zeros, (dst ^ (stage & 2) * BYTES) + (stage & 1) * BYTES + i * 1024);
        }
    }

    // subtile i (16 rows)
    __device__ __forceinline__ x8 read(int i, int stage) const {
        if constexpr (ROWS) {
            const int row = SPREAD ? 64 * (i >> 2) + 4 * (i & 3) : 16 * i;
            return *(__attribute__((address_space(3))) const x8*)(uintptr_t)(at[0] + stage * BYTES + row * 64);
        } else {
            typedef __attribute__((address_space(3))) s16x4 lds_s4;
            const uint32_t a = at[i] + stage * BYTES;
            const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)a);
            const s16x4 w = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)(a + 4 * RB));
            return __builtin_bit_cast(x8, __builtin_shufflevector(v, w, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

// A workgroup's tile is BM x BN, a wavefront's WM x WN in 16 x 16 subtiles, with four steps of 32 k in LDS. A step has two
// parts, each with half the wavefront's rows of A: a part's matrix instructions run while the next part's operands come
// from LDS. Between the parts every wavefront has read the whole step, so there is the one barrier: behind it the
// next step's first operands are read and the step four on is loaded into the stage that became free. A load has two and a half
// steps to arrive.
template <typename T, bool A_ROWS, bool B_ROWS, int EPILOGUE, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN), 2) void k_product(const ProductArgs q) {
    typedef typename Vec<T>::x8 x8;
    constexpr int WAVES = (BM / WM) * (BN / WN), IM = WM / 16, IN = WN / 16, HALF = IM / 2;
    typedef Tile<T, A_ROWS, EPILOGUE == LOGITS, BM, WAVES, IM> TA;
    typedef Tile<T, B_ROWS, false, BN, WAVES, IN> TB;
    constexpr int LOADS = TA::LOADS + TB::LOADS;
    __shared__ __attribute__((aligned(1024))) char smem[STAGES * (TA::BYTES + TB::BYTES)];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, lo = lane & 15, hi = lane >> 4;
    const int wm = wave / (BN / WN) * WM, wn = wave % (BN / WN) * WN;

    // Workgroups go round the eight XCDs in turn; each XCD gets a contiguous part of the tiles, in groups of four m by
    // all n, so that the workgroups that run together on it share operands in its L2.
    const int tiles = q.m_tiles * q.n_tiles * q.splits;
    const int xcd = blockIdx.x & 7, per = tiles >> 3, rest = tiles & 7;
    int id = xcd * per + (xcd < rest ? xcd : rest) + (blockIdx.x >> 3);
    const int split = id / (q.m_tiles * q.n_tiles);
    id -= split * (q.m_tiles * q.n_tiles);
    const int group = id / (4 * q.n_tiles), in_group = q.m_tiles - 4 * group < 4 ? q.m_tiles - 4 * group : 4;
    id -= group * 4 * q.n_tiles;
    const long m0 = (long)(4 * group + id % in_group) * BM, n0 = (long)(id / in_group) * BN;

    const long k0 = split * q.split_k, k1 = k0 + q.split_k < q.K ? k0 + q.split_k : q.K;
    const long K = k1 > k0 ? k1 - k0 : 0;
    const int steps = 2 * (int)((K + 2 * BK - 1) / (2 * BK));
    TA a;
    TB b;
    a.init(q.A, q.lda, q.M, m0, k0, (lds_char*)smem, wave, lane, wm);
    b.init(q.B, q.ldb, q.N, n0, k0, (lds_char*)smem + STAGES * TA::BYTES, wave, lane, wn);

    f32x4 c[IM][IN] = {};
    x8 fa0[HALF], fa1[HALF], fb0[IN], fb1[IN];
    // The last 64 k, the only ones that may be fewer, are steps 0 and 1, and k 32 (t - 2) on are step t: so the loop loads
    // whole steps only, and there is an even number of them.
    auto load_first = [&](int t) {
        const int k = steps - 2 + t;
        const long left = K - (long)BK * k;
        if (left >= BK) {
#pragma unroll
            for (int i = 0; i < TA::LOADS; ++i) a.load(k, t, i);
#pragma unroll
            for (int i = 0; i < TB::LOADS; ++i) b.load(k, t, i);
        } else {
            a.load_end(k, t, (int)left, q.zeros, wave, lane);
            b.load_end(k, t, (int)left, q.zeros, wave, lane);
        }
    };
    // Step t in stage ODD (0 or 1) of this turn; f: this step's part of B, g: where the next one's goes. Reads and loads
    // are spread over the subtile rows' instructions, and the fences keep that order. Behind the last step an old stage
    // is read once more, for nothing.
    auto step = [&](int t, auto odd, auto more, x8(&f)[IN], x8(&g)[IN]) {
        constexpr int ODD = decltype(odd)::value;
        constexpr bool LOAD = decltype(more)::value;   // step t + 4 is loaded
#pragma unroll
        for (int i = 0; i < HALF; ++i) {
            if (2 * i < HALF) {
                fa1[2 * i] = a.read(HALF + 2 * i, ODD);
                fa1[2 * i + 1] = a.read(HALF + 2 * i + 1, ODD);
            }
#pragma unroll
            for (int j = 0; j < IN; ++j) c[i][j] = Vec<T>::mfma(fa0[i], f[j], c[i][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
        // This wavefront has read the step and its loads of the next one have arrived (those of the two after it may be
        // under way); then everybody's.
        if constexpr (LOAD)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * LOADS) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        asm volatile("s_barrier" ::: "memory");
        if constexpr (ODD) {
            a.turn();
            b.turn();
        }
        constexpr int NEXT = ODD ? 0 : 1, FREE = ODD ? 3 : 0;
#pragma unroll
        for (int i = 0; i < HALF; ++i) {
#pragma unroll
            for (int j = 2 * i * IN / HALF; j < 2 * (i + 1) * IN / HALF && j < IN; ++j) g[j] = b.read(j, NEXT);
            if (2 * i >= HALF) {
                fa0[2 * i - HALF] = a.read(2 * i - HALF, NEXT);
                fa0[2 * i - HALF + 1] = a.read(2 * i - HALF + 1, NEXT);
            }
            if constexpr (LOAD) {
#pragma unroll
                for (int j = i * LOADS / HALF; j < (i + 1) * LOADS / HALF; ++j) {
                    if (j < TA::LOADS)
                        a.load(t + STAGES - 2, FREE, j);
                    else
                        b.load(t + STAGES - 2, FREE, j - TA::LOADS);
                }
            }
#pragma unroll
            for (int j = 0; j < IN; ++j) c[HALF + i][j] = Vec<T>::mfma(fa1[i], f[j], c[HALF + i][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    if (steps > 0) {
        load_first(0);
        load_first(1);
        if (steps > 2) {
#pragma unroll
            for (int t = 2; t < STAGES; ++t) {
#pragma unroll
                for (int i = 0; i < TA::LOADS; ++i) a.load(t - 2, t, i);
#pragma unroll
                for (int i = 0; i < TB::LOADS; ++i) b.load(t - 2, t, i);
            }
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 1) * LOADS) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        asm volatile("s_barrier" ::: "memory");
        // (scalar loads that are still under way would make the compiler wait for all LDS reads in every turn)
        __builtin_amdgcn_s_waitcnt(0xc07f);
#pragma unroll
        for (int j = 0; j < IN; ++j) fb0[j] = b.read(j, 0);
#pragma unroll
        for (int i = 0; i < HALF; ++i) fa0[i] = a.read(i, 0);
        int t = 0;
        for (; t + STAGES < steps; t += 2) {
            step(t, std::integral_constant<int, 0>{}, std::true_type{}, fb0, fb1);
            step(t + 1, std::integral_constant<int, 1>{}, std::true_type{}, fb1, fb0);
        }
        for (; t < steps; t += 2) {
            step(t, std::integral_constant<int, 0>{}, std::false_type{}, fb0, fb1);
            step(t + 1, std::integral_constant<int, 1>{}, std::false_type{}, fb1, fb0);
        }
    }

    // lane: row n = lo of C, elements m = 4 hi + 0..3 of each subtile (16 hi + 0..15 of four subtiles where SPREAD)
    if constexpr (EPILOGUE == LOGITS) {
        const long first = m0 + wm + 16 * hi;   // of the lane's columns; each group of four subtiles is 64 on
        if (m0 + wm + WM > q.M) {               // columns past the vocabulary
#pragma unroll
            for (int i = 0; i < IM; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool out = first + 64 * (i >> 2) + 4 * (i & 3) + r >= q.M;
#pragma unroll
                    for (int j = 0; j < IN; ++j) c[i][j][r] = out ? -INFINITY : c[i][j][r];
                }
        }
#pragma unroll
        for (int j = 0; j < IN; ++j) {
            const long n = n0 + wn + 16 * j + lo;
            float m = -INFINITY;
#pragma unroll
            for (int i = 0; i < IM; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) m = nan_max(m, c[i][j][r]);
            m = nan_max(m, __shfl_xor(m, 16));
            m = nan_max(m, __shfl_xor(m, 32));
            const float top = m == -INFINITY ? 0.0f : m;
            const long tgt = n < q.N ? q.target[n] - first : -1;
            if (tgt >= 0 && tgt < 64 * (IM / 4) && (tgt & 63) < 16 && first + tgt < q.M) {
                const int k = (int)tgt;
                float z = 0.0f;
#pragma unroll
                for (int i = 0; i < IM; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) z = k == 64 * (i >> 2) + 4 * (i & 3) + r ? c[i][j][r] : z;
                q.zt[n] = z;
            }
            float sum = 0.0f;
#pragma unroll
            for (int g = 0; g < IM / 4; ++g) {
                T e[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float v = exp_of(c[4 * g + i / 4][j][i & 3] - top);
                    sum += v;
                    e[i] = (T)v;
                }
                const long v = first + 64 * g;
                if (q.p != nullptr && n < q.N && v < q.ldp) {
                    T* to = (T*)q.p + n * q.ldp + v;
                    *(x8*)to = *(const x8*)e;
                    *(x8*)(to + 8) = *(const x8*)(e + 8);
                }
            }
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (hi == 0 && n < q.N && m0 + wm < q.M) q.stat[n * q.segs + (m0 + wm) / WM] = make_float2(m, sum);
        }
    } else {
        const float alpha = q.acc == nullptr ? *q.alpha : 1.0f;
#pragma unroll
        for (int j = 0; j < IN; ++j) {
            const long n = n0 + wn + 16 * j + lo;
#pragma unroll
            for (int i = 0; i < IM; ++i) {
                const long m = m0 + wm + 16 * i + 4 * hi;
                if (n >= q.N || m >= q.M) continue;
                f32x4 v = c[i][j];
                if (q.acc != nullptr) {
                    f32x4* to = (f32x4*)(q.acc + (split * q.N + n) * q.ldacc + m);
                    if (q.add) v += *to;
                    *to = v;
                    continue;
                }
                T* to = (T*)q.C + n * q.ldc + m;
                T e[4] = {(T)(v[0] * alpha), (T)(v[1] * alpha), (T)(v[2] * alpha), (T)(v[3] * alpha)};
                if (q.vector) {
                    *(uint2*)to = *(const uint2*)e;
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (m + r < q.M) to[r] = e[r];
                }
            }
        }
    }
}

// C = alpha times the sum of the splits' parts, in their order
template <typename T>
__global__ __launch_bounds__(256) void k_join(const float* acc, int splits, long rows, long M, long Mp, void* C, const float* alpha) {
    const long n = rows * Mp / 4;
    const float a = *alpha;
    for (long i = blockIdx.x * 256l + threadIdx.x; i < n; i += 256l * gridDim.x) {
        f32x4 v = ((const f32x4*)acc)[i];
        for (int s = 1; s < splits; ++s) v += ((const f32x4*)acc)[s * n + i];
        const long row = 4 * i / Mp, m = 4 * i - row * Mp;
        T* to = (T*)C + row * M + m;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (m + r < M) to[r] = (T)(v[r] * a);
    }
}

// a token's weight: 0 where it is ignored, NaN where its target is no column
__device__ __forceinline__ float weight_of(long target, long ignore, long V, const float* row_weight, long i) {
    if (target == ignore) return 0.0f;
    if (target < 0 || target >= V) return NAN;
    return row_weight == nullptr ? 1.0f : row_weight[i];
}

struct Scalars {
    uint32_t zeros[4];
    float alpha;    // what dx and dW are multiplied by
    float per;      // what the sum of the losses is multiplied by
    float w_scale;  // G holds the weights times this (a power of 2: the largest weight to [1, 2))
};

// counts the tokens that are not ignored; one workgroup
__global__ __launch_bounds__(1024) void k_prepare(const long* target, long N, long ignore, int mean, const float* row_weight,
                                                  const float* grad_scale, float g, Scalars* out) {
    __shared__ int slot[16];
    __shared__ float most[16];
    int count = 0;
    float w = 0.0f;
    for (long i = threadIdx.x; i < N; i += 1024) {
        const bool kept = target[i] != ignore;
        count += kept;
        if (kept && row_weight != nullptr) {
            const float a = fabsf(row_weight[i]);
            if (a < INFINITY) w = fmaxf(w, a);
        }
    }
    count = reduce_threads<1024, Sum>(count, slot);
    w = reduce_threads<1024, NanMax>(w, most);
    if (threadIdx.x == 0) {
        const float per = mean ? 1.0f / (float)(count > 0 ? count : 1) : 1.0f;
        float s = 1.0f;
        if (w > 0.0f) s = ldexpf(1.0f, -min(max(ilogbf(w), -100), 100));
        for (int i = 0; i < 4; ++i) out->zeros[i] = 0;
        out->per = per;
        out->w_scale = s * g;
        out->alpha = per * (grad_scale == nullptr ? 1.0f : *grad_scale) / (s * g);
    }
}

struct FinishArgs {
    long V, segs, ldp, ignore;
    int seg;                     // columns of a segment, 2^seg
    const long* target;
    const float *row_weight, *zt;
    const float2* stat;
    void* p;                     // or null: the loss alone
    float *loss, *lse;
    const Scalars* scal;
};

// one token a blockIdx.x: lse from the segments' statistics, the loss, and p -> G in the columns of blockIdx.y
template <typename T>
__global__ __launch_bounds__(256) void k_finish(const FinishArgs q) {
    __shared__ float slot[4];
    const long i = blockIdx.x;
    const float2* stat = q.stat + i * q.segs;
    float m = -INFINITY;
    for (long s = threadIdx.x; s < q.segs; s += 256) m = nan_max(m, stat[s].x);
    m = reduce_threads<256, NanMax>(m, slot);
    float sum = 0.0f;
    for (long s = threadIdx.x; s < q.segs; s += 256) sum += stat[s].y * exp_of(stat[s].x - m);
    sum = reduce_threads<256, Sum>(sum, slot);
    const float lse = m + logf(sum);
    const long t = q.target[i];
    const float w = weight_of(t, q.ignore, q.V, q.row_weight, i);
    const bool in = t >= 0 && t < q.V && t != q.ignore;
    const float d = in ? q.zt[i] - lse : w;   // log of the target's probability (or 0, or NaN)
    if (blockIdx.y == 0 && threadIdx.x == 0) {
        q.loss[i] = w == 0.0f ? 0.0f : -w * d;
        if (q.lse != nullptr) q.lse[i] = lse;
    }
    if (q.p == nullptr) return;
    T* p = (T*)q.p + i * q.ldp;
    const float f = w * q.scal->w_scale;
    for (long v = 8l * (threadIdx.x + 256l * blockIdx.y); v < q.ldp; v += 8l * 256 * gridDim.y) {
        float e[8];
        if (w == 0.0f) {
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] = 0.0f;
        } else {
            load8(p + v, 8, e);
            const float s = v < q.V ? f * exp_of(stat[v >> q.seg].x - lse) : 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] = v + k < q.V ? e[k] * s : 0.0f;
            if (in && t >= v && t < v + 8) {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (t == v + k) e[k] = f * expm1f(d);
            }
        }
        store8(p + v, 8, e);
    }
}

// the sum (or mean) of the tokens' losses; one workgroup, a fixed order
__global__ __launch_bounds__(1024) void k_total(const float* loss, long N, const Scalars* scal, float* out) {
    __shared__ double slot[16];
    double sum = 0.0;
    for (long i = threadIdx.x; i < N; i += 1024) sum += (double)loss[i];
    sum = reduce_threads<1024, Sum>(sum, slot);
    if (threadIdx.x == 0) *out = (float)(sum * (double)scal->per);
}

// rows of H elements to rows of Hp (the next multiple of 8), the rest 0: operands whose rows do not start on 16 bytes
template <typename T>
__global__ __launch_bounds__(256) void k_pad(const T* src, long ld, long rows, long H, long Hp, T* dst) {
    const long pieces = Hp / 8;
    for (long i = blockIdx.x * 256l + threadIdx.x; i < rows * pieces; i += 256l * gridDim.x) {
        const long row = i / pieces, at = 8 * (i - row * pieces);
        float v[8];
        load8(src + row * ld + at, H - at >= 8 ? 8 : (int)(H - at), v);
        store8(dst + row * Hp + at, 8, v);
    }
}

constexpr long MAX_N = 1l << 31, MAX_HV = 1l << 22;   // 256 rows stay within 32-bit byte offsets

long up(long v, long to) { return (v + to - 1) / to * to; }
long over(long v, long by) { return (v + by - 1) / by; }

// the workgroup tiles: 256 x 256 for eight wavefronts, 128 x 128 and 128 (m) x 64 (n) for four
enum { BIG, MID, NARROW };
constexpr int TILE_M[] = {256, 128, 128}, TILE_N[] = {256, 128, 64};
constexpr int SLOTS[] = {256, 512, 768};        // workgroups the device holds at once
constexpr double STEP_US[] = {1.8, 1.1, 0.8};   // 64 k of a full device

struct Shape {
    int kind;
    long m_tiles, n_tiles;
    int splits;
    long split_k;
};

// microseconds of C [N][M] over K in tiles of `kind`, in `splits` parts of K
double time_of(int kind, long M, long N, long K, long splits) {
    const double rounds = (double)over(over(M, TILE_M[kind]) * over(N, TILE_N[kind]) * splits, SLOTS[kind]);
    const double join = splits > 1 ? 4.0 + 8.0 * (double)(M * N * splits) / 4e6 : 0.0;
    return rounds * (STEP_US[kind] * (double)over(over(K, 64), splits) + 2.0) + join;
}

// rows of fp32 sums that dx over several parts of K may take. Like all of the workspace it does not shrink with more
// tokens, so that what fits for some fits for fewer.
long split_rows(long tokens) {
    const long most = 2 * tokens > 16384 ? 2 * tokens : 16384;
    return 64 * tokens < most ? 64 * tokens : most;
}

// the fastest by time_of, in at most `most` parts of K
Shape shape_of(long M, long N, long K, long most) {
    Shape best = {};
    double least = 1e300;
    for (int kind = BIG; kind <= NARROW; ++kind)
        for (long splits = 1; splits <= most && (splits == 1 || over(K, 64) >= 4 * splits); ++splits) {
            const double t = time_of(kind, M, N, K, splits);
            if (t < least * 0.98) {
                least = t;
                best = {kind, over(M, TILE_M[kind]), over(N, TILE_N[kind]), (int)splits, 64 * over(over(K, 64), splits)};
            }
        }
    return best;
}

// where things lie in the workspace, for `tokens` tokens at a time
struct Layout {
    long scal, loss, zt, stat, p, dx_acc, dw_acc, x, w, bytes;
    long segs, ldp, Hp;
    Shape logits, dx;            // of a full piece of the tokens
};
Layout layout_of(long N, long H, long V, int grads, bool pad, long tokens) {
    Layout l;
    l.logits = shape_of(V, tokens, H, 1);
    l.dx = shape_of(H, tokens, V, tokens > 0 ? split_rows(tokens) / tokens : 1);
    l.segs = over(V, TILE_M[l.logits.kind] / 2);
    l.ldp = up(V, 64);
    l.Hp = up(H, 8);
    long at = 0;
    auto take = [&](long bytes) {
        const long was = at;
        at += up(bytes, 256);
        return was;
    };
    l.scal = take(sizeof(Scalars));
    l.loss = take(4 * N);
    l.zt = take(4 * tokens);
    l.stat = take(8 * tokens * over(V, 64));
    l.p = take(grads ? 2 * tokens * l.ldp : 0);
    l.dx_acc = take((grads & 1) ? 4 * split_rows(tokens) * l.Hp : 0);
    l.dw_acc = take((grads & 2) && tokens < N ? 4 * l.Hp * V : 0);
    l.x = take(pad ? 2 * N * l.Hp : 0);
    l.w = take(pad ? 2 * V * l.Hp : 0);
    l.bytes = at;
    return l;
}

// most tokens at a time within `most` bytes: all, or a multiple of 256 (at least 256)
long tokens_of(long N, long H, long V, int grads, bool pad, long most) {
    if (N <= 256 || layout_of(N, H, V, grads, pad, N).bytes <= most) return N;
    long lo = 1, hi = over(N, 256);   // in units of 256: lo is taken, hi is too many
    while (hi - lo > 1) {
        const long mid = (lo + hi) / 2;
        if (layout_of(N, H, V, grads, pad, 256 * mid).bytes <= most)
            lo = mid;
        else
            hi = mid;
    }
    // the pieces alike
    const long pieces = over(N, 256 * lo), even = up(over(N, pieces), 256);
    return even < 256 * lo ? even : 256 * lo;
}

int check_sizes(int type, long N, long H, long V) {
    if (type != SPANQR_BF16 && type != SPANQR_FP16)
        return error(SPANQR_EINVAL, "linear_cross_entropy: x and W are bf16 or fp16");
    if (N < 0 || N > MAX_N || H < 1 || H > MAX_HV || V < 1 || V > MAX_HV)
        return error(SPANQR_EINVAL, "linear_cross_entropy: N = %ld, H = %ld, V = %ld", N, H, V);
    return SPANQR_OK;
}

// whether an operand is copied to rows that start on 16 bytes
bool needs_pad(const void* x, long ldx, const void* w, long ldw, long H) {
    return H % 8 != 0 || ldx % 8 != 0 || ldw % 8 != 0 || (uintptr_t)x % 16 != 0 || (uintptr_t)w % 16 != 0 ||
           ldx > MAX_HV || ldw > MAX_HV;
}

struct Call {
    int mean;
    bool reduced, pad;
    long N, H, V;
    const void *x, *w;
    long ldx, ldw;
    const long* target;
    long ignore;
    const float *row_weight, *grad_scale;
    float *loss, *lse;
    void *dx, *dw;
};

template <typename T, bool A_ROWS, bool B_ROWS, int EPILOGUE>
void product(const Shape& s, ProductArgs q, hipStream_t st) {
    q.m_tiles = (int)s.m_tiles, q.n_tiles = (int)s.n_tiles, q.splits = s.splits, q.split_k = s.split_k;
    const unsigned grid = (unsigned)(s.m_tiles * s.n_tiles * s.splits);
    if (s.kind == BIG)
        k_product<T, A_ROWS, B_ROWS, EPILOGUE, 256, 256, 128, 64><<<grid, 512, 0, st>>>(q);
    else if (s.kind == MID)
        k_product<T, A_ROWS, B_ROWS, EPILOGUE, 128, 128, 64, 64><<<grid, 256, 0, st>>>(q);
    else
        k_product<T, A_ROWS, B_ROWS, EPILOGUE, 128, 64, 64, 32><<<grid, 256, 0, st>>>(q);
}

template <typename T>
int enqueue(const Call& c, char* ws, long tokens, hipStream_t st) {
    const int grads = (c.dx != nullptr ? 1 : 0) | (c.dw != nullptr ? 2 : 0);
    const Layout l = layout_of(c.N, c.H, c.V, grads, c.pad, tokens);
    Scalars* scal = (Scalars*)(ws + l.scal);
    float* loss = c.reduced ? (float*)(ws + l.loss) : c.loss;
    const T *x = (const T*)c.x, *w = (const T*)c.w;
    long ldx = c.ldx, ldw = c.ldw;
    k_prepare<<<1, 1024, 0, st>>>(c.target, c.N, c.ignore, c.mean, c.row_weight, c.grad_scale, g_scale<T>(), scal);
    if (c.pad) {
        auto grid = [&](long rows) { return (unsigned)(over(rows * l.Hp / 8, 256) < 4096 ? over(rows * l.Hp / 8, 256) : 4096); };
        if (c.N > 0) k_pad<T><<<grid(c.N), 256, 0, st>>>(x, ldx, c.N, c.H, l.Hp, (T*)(ws + l.x));
        k_pad<T><<<grid(c.V), 256, 0, st>>>(w, ldw, c.V, c.H, l.Hp, (T*)(ws + l.w));
        x = (const T*)(ws + l.x), w = (const T*)(ws + l.w);
        ldx = ldw = l.Hp;
    }
    ProductArgs base = {};
    base.zeros = scal->zeros;
    base.ldp = l.ldp, base.segs = l.segs;
    base.ldc = c.H, base.ldacc = l.Hp;
    base.alpha = &scal->alpha;
    // no tokens: dW is a product over nothing
    for (long at = 0; at < c.N || (at == 0 && c.dw != nullptr); at += tokens > 0 ? tokens : 1) {
        const long n = c.N - at < tokens ? c.N - at : tokens;
        if (n > 0) {
            ProductArgs q = base;
            q.M = c.V, q.N = n, q.K = l.Hp;
            q.A = w, q.lda = ldw;
            q.B = x + at * ldx, q.ldb = ldx;
            q.target = c.target + at;
            q.zt = (float*)(ws + l.zt);
            q.stat = (float2*)(ws + l.stat);
            q.p = grads ? ws + l.p : nullptr;
            Shape s = l.logits;
            s.n_tiles = over(n, TILE_N[s.kind]);
            product<T, true, true, LOGITS>(s, q, st);
            FinishArgs f = {c.V, l.segs, l.ldp, c.ignore, s.kind == BIG ? 7 : 6, c.target + at,
                            c.row_weight == nullptr ? nullptr : c.row_weight + at, q.zt, q.stat, q.p, loss + at,
                            c.lse == nullptr ? nullptr : c.lse + at, scal};
            const long split = grads ? (n >= 2048 ? 1 : 2048 / n) : 1, most = over(l.ldp, 2048);
            k_finish<T><<<dim3((unsigned)n, (unsigned)(split < most ? split : most)), 256, 0, st>>>(f);
        }
        if (c.dx != nullptr && n > 0) {
            ProductArgs d = base;
            d.M = c.H, d.N = n, d.K = c.V;
            d.A = w, d.lda = ldw;
            d.B = ws + l.p, d.ldb = l.ldp;
            T* C = (T*)c.dx + at * c.H;
            d.C = C;
            d.vector = c.H % 4 == 0 && (uintptr_t)C % 8 == 0;
            d.acc = l.dx.splits > 1 ? (float*)(ws + l.dx_acc) : nullptr;
            Shape s = l.dx;
            s.n_tiles = over(n, TILE_N[s.kind]);
            product<T, false, true, OUT>(s, d, st);
            if (d.acc != nullptr)
                k_join<T><<<2048, 256, 0, st>>>(d.acc, s.splits, n, c.H, l.Hp, C, &scal->alpha);
        }
        if (c.dw != nullptr) {
            ProductArgs d = base;
            d.M = c.H, d.N = c.V, d.K = n;
            d.A = x + at * ldx, d.lda = ldx;
            d.B = ws + l.p, d.ldb = l.ldp;
            d.C = c.dw;
            d.vector = c.H % 4 == 0 && (uintptr_t)c.dw % 8 == 0;
            d.acc = tokens < c.N ? (float*)(ws + l.dw_acc) : nullptr;
            d.add = at > 0;
            product<T, false, false, OUT>(shape_of(c.H, c.V, n, 1), d, st);
            if (d.acc != nullptr && at + n == c.N)
                k_join<T><<<2048, 256, 0, st>>>(d.acc, 1, c.V, c.H, l.Hp, c.dw, &scal->alpha);
        }
    }
    if (c.reduced) k_total<<<1, 1024, 0, st>>>(loss, c.N, scal, c.loss);
    return launched("linear_cross_entropy");
}

}  // namespace

extern "C" {

long spanqr_linear_cross_entropy_workspace(int type, long N, long H, long V, int grads, long most_bytes) {
    const int rc = check_sizes(type, N, H, V);
    if (rc != SPANQR_OK) return rc;
    // (with room for the copies that unaligned operands need)
    return layout_of(N, H, V, grads, true, tokens_of(N, H, V, grads, true, most_bytes)).bytes;
}

int spanqr_linear_cross_entropy(int type, int reduction, long N, long H, long V, const void* x, long ldx, const void* w,
                                long ldw, const long* target, long ignore_index, const float* row_weight,
                                const float* grad_scale, float* loss, float* lse, void* dx, void* dw, void* workspace,
                                long workspace_bytes, void* stream) {
    const int rc = check_sizes(type, N, H, V);
    if (rc != SPANQR_OK) return rc;
    if (reduction != SPANQR_REDUCE_NONE && reduction != SPANQR_REDUCE_SUM && reduction != SPANQR_REDUCE_MEAN)
        return error(SPANQR_EINVAL, "linear_cross_entropy: unknown reduction %d", reduction);
    const bool reduced = reduction != SPANQR_REDUCE_NONE;
    if ((N > 0 && (x == nullptr || target == nullptr)) || w == nullptr || workspace == nullptr ||
        (loss == nullptr && (N > 0 || reduced)))
        return error(SPANQR_EINVAL, "linear_cross_entropy: a missing pointer");
    if ((N > 1 && ldx < H) || (V > 1 && ldw < H))
        return error(SPANQR_EINVAL, "linear_cross_entropy: a row stride below H");
    const int grads = (dx != nullptr ? 1 : 0) | (dw != nullptr ? 2 : 0);
    const bool pad = needs_pad(x, N > 1 ? ldx : 0, w, V > 1 ? ldw : 0, H);
    const long tokens = tokens_of(N, H, V, grads, pad, workspace_bytes), need = layout_of(N, H, V, grads, pad, tokens).bytes;
    if (need > workspace_bytes) return error(SPANQR_EINVAL, "linear_cross_entropy: the workspace needs %ld bytes", need);
    const Call c = {reduction == SPANQR_REDUCE_MEAN, reduced, pad, N, H, V, x, w, ldx, ldw, target, ignore_index,
                    row_weight, grad_scale, loss, lse, dx, dw};
    hipStream_t st = (hipStream_t)stream;
    return type == SPANQR_BF16 ? enqueue<bf16>(c, (char*)workspace, tokens, st)
                               : enqueue<fp16>(c, (char*)workspace, tokens, st);
}

}  // extern "C"
