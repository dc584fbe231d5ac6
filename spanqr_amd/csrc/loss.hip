// loss.hip -- softmax cross entropy over a large vocabulary from the hidden states and the head's weights, without
// keeping the logits, and its gradients.
//
//   z = x W^T [N, V],  lse_i = log sum_j exp z_ij,  loss_i = w_i (lse_i - z_i,t_i)      (w_i = 0 where t_i is ignored)
//   G_ij = w_i (exp(z_ij - lse_i) - [j = t_i]),  dx = a G W,  dW = a G^T x      (a = 1, or 1 / tokens that count)
//
// Three products of 2 N H V operations each. The product of the logits ends in its own softmax statistics: for 64 or
// 128 neighbouring columns of a token it leaves the maximum m and the sum of exp(z - m), and, where gradients are wanted,
// the exponentials p = exp(z - m) themselves, rounded to the 16-bit type once. The target's column is left out of all
// three and its logit kept: with R the sum over the others of exp(z_ij - z_i,t) the loss is log1p R, within 1e-6 of itself
// also where the token is sure (next to the target's 1 a sum would lose R). One pass over p turns it into G (times
// exp(m - lse); the target's element from the loss), and G goes into the other two products. So nothing is multiplied
// twice, and what is held is 16 bits an element for as many tokens at a time as the workspace takes. The gradients' error
// is then that of G's elements, rounded twice, and of one rounding at the end: 1.0 to 1.3 times the error of a result that
// is rounded at the end alone where many elements add up, up to 1.7 (three roundings) where one makes a gradient; 1.0
// times for up to 32 tokens, whose p and G keep what is rounded off. A G in fp32 would take the products' rate.
#include <limits.h>
#include <math.h>

#include <algorithm>
#include <type_traits>
#include <utility>

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

template <typename T>
struct Vec;
template <>
struct Vec<bf16> {
    typedef bf16x8 x8;
};
template <>
struct Vec<fp16> {
    typedef fp16x8 x8;
};

// c += a b, 16 x 16 x 32. In inline asm, because c has to stay where it is: the compiler moves accumulators about
// between registers when they fill half the file. ACC: c in accumulation registers. It does not know that these are
// matrix instructions, whose results may not be read for up to 18 clocks, and may copy c as soon as a loop ends: so the
// loop's last one waits (LAST; the matrix pipe is busy with it for most of that time), in the same piece of asm.
#define SPANQR_MFMA(OP, AT, WAIT)                                                               \
    asm volatile("v_mfma_f32_16x16x32_" OP " %0, %1, %2, %0" WAIT : "+" AT(c) : "v"(a), "v"(b))
#define SPANQR_MFMA_WAIT "\n\ts_nop 15\n\ts_nop 3"
// The same, and behind it 16 bytes a lane from base + off to LDS at `lds` + IMM + 16 lane, asynchronously (counted by
// vmcnt). The load too is in inline asm because the compiler would wait for it before any later LDS read; it has no
// register output. The matrix instruction fills the wait between m0 and its use.
#define SPANQR_MFMA_LOAD(OP, AT)                                                                 \
    asm volatile("s_add_u32 m0, %5, %6\n\tv_mfma_f32_16x16x32_" OP " %0, %1, %2, %0\n\t"         \
                 "global_load_lds_dwordx4 %3, %4"                                                \
                 : "+" AT(c)                                                                     \
                 : "v"(a), "v"(b), "v"(off), "s"(base), "s"(lds), "n"(IMM)                       \
                 : "memory", "scc")
template <typename T, bool ACC, bool LAST>
__device__ __forceinline__ void mfma(typename Vec<T>::x8 a, typename Vec<T>::x8 b, f32x4& c) {
    if constexpr (std::is_same<T, bf16>::value) {
        if constexpr (ACC && LAST)
            SPANQR_MFMA("bf16", "a", SPANQR_MFMA_WAIT);
        else if constexpr (ACC)
            SPANQR_MFMA("bf16", "a", "");
        else if constexpr (LAST)
            SPANQR_MFMA("bf16", "v", SPANQR_MFMA_WAIT);
        else
            SPANQR_MFMA("bf16", "v", "");
    } else {
        if constexpr (ACC && LAST)
            SPANQR_MFMA("f16", "a", SPANQR_MFMA_WAIT);
        else if constexpr (ACC)
            SPANQR_MFMA("f16", "a", "");
        else if constexpr (LAST)
            SPANQR_MFMA("f16", "v", SPANQR_MFMA_WAIT);
        else
            SPANQR_MFMA("f16", "v", "");
    }
}
template <typename T, bool ACC, int IMM>
__device__ __forceinline__ void mfma_load(typename Vec<T>::x8 a, typename Vec<T>::x8 b, f32x4& c, const void* base, uint32_t off,
                                          uint32_t lds) {
    if constexpr (std::is_same<T, bf16>::value) {
        if constexpr (ACC)
            SPANQR_MFMA_LOAD("bf16", "a");
        else
            SPANQR_MFMA_LOAD("bf16", "v");
    } else {
        if constexpr (ACC)
            SPANQR_MFMA_LOAD("f16", "a");
        else
            SPANQR_MFMA_LOAD("f16", "v");
    }
}

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
    float2* stat;                // [token][segs]: maximum (-inf: no logit), sum of the exponentials
    long segs;
    void* p;                     // exponentials [token][ldp], or null
    long ldp;
    // dx, dW
    void* C;
    long ldc;
    int vector;                  // C takes 16-byte stores
    float* acc;                  // fp32 sums [split][N][ldacc], or null: C directly
    long ldacc;
    int add;                     // add to what acc holds
    const float* alpha;
};

enum { LOGITS, OUT };

typedef __attribute__((address_space(3))) char lds_char;
typedef short s16x4 __attribute__((ext_vector_type(4)));

// 16 bytes a lane from base + off to LDS at `lds` + 16 lane, asynchronously
__device__ __forceinline__ void load_lds(const void* base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory");
}
__device__ __forceinline__ void load_lds_any(const void* at, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(at) : "memory");
}

constexpr int BK = 64;               // k of a step; two steps are in LDS

// One operand's tiles of R rows (m or n) by 64 k in LDS, and the way there and into registers.
// ROWS (k neighbours in memory): R rows of 128 bytes; the 16-byte chunk c of a row lies at c ^ swizzle(row), so that the
// 16 rows a matrix instruction reads spread over the banks. LDS serves lanes 0-3, 12-15, 20-27 of each 32 together and
// then the others: the swizzle gives each of those sixteen a slot of its own among 256 bytes (a read then takes 4
// clocks; 8 with swizzle(row) = row % 8).
// Otherwise (m or n neighbours): 64 k-rows of 2 R bytes, read by the transposing LDS read (16 lanes fetch 4 k-rows of
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
    long step;                   // bytes for 64 k
    uint32_t off[LOADS];
    uint32_t dst;                // LDS of the wavefront's first load into this step's buffer
    uint32_t at[ROWS ? 2 : SUB]; // LDS of the lane's fragments in this step's buffer

    __device__ __forceinline__ static int swizzle(int i) {   // of a row, or of a k
        if constexpr (ROWS) {
            const int u = SPREAD ? (i >> 4 & 3) << 1 | (i >> 1 & 1) : i >> 1 & 7;
            return ((u >> 2 ^ u >> 1) & 1) << 2 | (u >> 2) << 1 | (u & 1);
        } else {
            return R >= 256 ? (i & 3) | (i >> 3 & 3) << 2 : R == 128 ? (i & 3) | (i >> 3 & 1) << 2 : (i >> 1 & 1) | (i >> 3 & 1) << 1;
        }
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
                const int row = 8 * (wave * LOADS + i) + (lane >> 3);
                const int r = (int)(r0 + row < rows ? row : rows - 1 - r0);   // rows past the end: any, not used
                off[i] = (uint32_t)(2 * r) * (uint32_t)ld + 16 * ((lane & 7) ^ swizzle(row));
            }
            const int row = SPREAD ? 16 * (lo >> 2) + (lo & 3) : lo;
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) at[ks] = lds0 + (first + row) * 128 + 16 * ((4 * ks + hi) ^ swizzle(row));
        } else {
            base = (const char*)src + 2 * (r0 + k0 * ld);
            step = 2 * BK * ld;
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int k = (wave * LOADS + i) * PER + lane / LPR, c = lane % LPR;
                int col = 16 * ((c >> 1) ^ swizzle(k)) + 8 * (c & 1);
                if (r0 + col >= rows) col = 0;
                off[i] = (uint32_t)(2 * k) * (uint32_t)ld + 2 * col;
            }
            const int k = 8 * hi + (lo >> 2);
#pragma unroll
            for (int i = 0; i < SUB; ++i)
                at[i] = lds0 + k * RB + (((first / 16 + i) ^ swizzle(k)) << 5) + 8 * (lo & 3);
        }
    }

    // to the other buffer (the bit is clear in every address: each operand's buffers start on a multiple of both)
    __device__ __forceinline__ void turn() {
        dst ^= BYTES;
#pragma unroll
        for (int i = 0; i < (ROWS ? 2 : SUB); ++i) at[i] ^= BYTES;
    }

    // instruction i of the load of k 64 t on into this step's buffer (other = 0) or the other one (BYTES)
    __device__ __forceinline__ void load(int t, int other, int i) const { load_lds(base + t * step, off[i], (dst ^ other) + i * 1024); }

    // all of the load of k 64 t on into this step's buffer where only `left` k are left
    __device__ __forceinline__ void load_end(int t, int left, const void* zeros, int wave, int lane) const {
        const char* b = base + t * step;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            int k;
            if constexpr (ROWS)
                k = 8 * ((lane & 7) ^ swizzle(8 * (wave * LOADS + i) + (lane >> 3)));
            else
                k = (wave * LOADS + i) * PER + lane / LPR;
            load_lds_any(k < left ? (const void*)(b + off[i]) : zeros, dst + i * 1024);
        }
    }

    // from here on every load reads the same 16 bytes
    __device__ __forceinline__ void stay(const void* at16) {
        base = (const char*)at16;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) off[i] = 0;
    }

    // subtile i (16 rows), k 32 ks to 32 ks + 31 of this step
    __device__ __forceinline__ x8 read(int i, int ks) const {
        if constexpr (ROWS) {
            const int row = SPREAD ? 64 * (i >> 2) + 4 * (i & 3) : 16 * i;
            return *(__attribute__((address_space(3))) const x8*)(uintptr_t)(at[ks] + row * 128);
        } else {
            typedef __attribute__((address_space(3))) s16x4 lds_s4;
            const uint32_t a = at[i] + ks * 32 * RB;
            const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)a);
            const s16x4 w = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)(a + 4 * RB));
            return __builtin_bit_cast(x8, __builtin_shufflevector(v, w, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

template <int... I, typename F>
__device__ __forceinline__ void each(std::integer_sequence<int, I...>, F f) {
    (f(std::integral_constant<int, I>{}), ...);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// over the four rows of 16 lanes of a wavefront, lane for lane, without going through LDS
template <typename OP>
__device__ __forceinline__ float reduce_rows(float v, OP op) {
    auto both = [&](auto swapped) {
        const uint32_t a = swapped[0], b = swapped[1];   // (a bit_cast of a vector's element takes the first one)
        return op(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
    };
    uint32_t u = __builtin_bit_cast(uint32_t, v);
    u = __builtin_bit_cast(uint32_t, both(__builtin_amdgcn_permlane16_swap(u, u, false, false)));
    return both(__builtin_amdgcn_permlane32_swap(u, u, false, false));
}

// A group of a token's columns with maximum m has the exponentials 2^(z log2 e - top), top = m log2 e rounded: one fma for
// each. They are exp(z - m) 2^off, off being what top's rounding leaves: below 2^-7. Where m is larger (up to where
// m log2 e overflows), and where it is -inf (no logit: k_finish passes the group by), they are 2^((z - sub) log2 e). That
// form for all would cost the logits of 4000 x 1024 x 50257 7 us of 465.
struct Base {
    float sub, top;
};
__device__ __forceinline__ bool within(float m) { return fabsf(m) < 65536.0f; }
__device__ __forceinline__ Base base_of(float m) {
    return within(m) ? Base{0.0f, m * LOG2E} : Base{m == -INFINITY ? 0.0f : m, 0.0f};
}
__device__ __forceinline__ float off_of(float m) { return within(m) ? fmaf(m, LOG2E, -(m * LOG2E)) : 0.0f; }

// A workgroup's tile is BM x BN, each of its four wavefronts' WM x WN in 16 x 16 subtiles. A step of 64 k has two
// halves: while one half's matrix instructions run, the other half's operands come from LDS, in its first rows. Between
// the halves every wavefront has read the whole step, so there is the one barrier: behind it the next step's first half is
// read and the step after that is loaded into the buffer that became free.
// A 128 x 128 part for each wavefront (one per SIMD) reads LDS least: 64 KB for 64 matrix instructions a SIMD and 32 k,
// where eight wavefronts of 128 x 64 read 96 (8.6 / 8.0 / 8.65 ms for the three products of the size below, when four
// took 8.1 / 8.1 / 8.3).
// Bound by the matrix pipe and the clock that it leaves (1.7 to 1.85 GHz under this load): logits, dx and dW of
// 8192 x 5120 x 128000 in 7.9, 8.15 and 8.3 ms, 1290 to 1360 TFLOP/s; with a short k by what surrounds the loop, the first
// loads and the epilogue: 4000 x 1024 x 50257 in 465, 350 and 390 us, 890 to 1180 TFLOP/s.
template <typename T, bool A_ROWS, bool B_ROWS, int EPILOGUE, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(256, BM == 256 ? 1 : 2) void k_product(const ProductArgs q) {
    typedef typename Vec<T>::x8 x8;
    constexpr int WAVES = (BM / WM) * (BN / WN), IM = WM / 16, IN = WN / 16;
    static_assert(WAVES == 4, "");
    typedef Tile<T, A_ROWS, EPILOGUE == LOGITS, BM, WAVES, IM> TA;
    typedef Tile<T, B_ROWS, false, BN, WAVES, IN> TB;
    constexpr int LOADS = TA::LOADS + TB::LOADS;
    __shared__ __attribute__((aligned(1024))) char smem[2 * (TA::BYTES + TB::BYTES)];
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
    const int steps = K > 0 ? (int)((K + BK - 1) / BK) : 1;   // (without k one step of zeros)
    TA a;
    TB b;
    a.init(q.A, q.lda, q.M, m0, k0, (lds_char*)smem, wave, lane, wm);
    b.init(q.B, q.ldb, q.N, n0, k0, (lds_char*)smem + 2 * TA::BYTES, wave, lane, wn);

    f32x4 c[IM][IN] = {};
    x8 fa[2][IM], fb[2][IN];
    // The last 64 k, the only ones that may be fewer, are step 0, and k 64 (t - 1) on are step t: so the loop loads whole
    // steps only.
    auto load_first = [&] {
        const int t = steps - 1, left = (int)(K - (long)BK * t);
        if (left == BK) {
#pragma unroll
            for (int i = 0; i < TA::LOADS; ++i) a.load(t, 0, i);
#pragma unroll
            for (int i = 0; i < TB::LOADS; ++i) b.load(t, 0, i);
        } else {
            a.load_end(t, left, q.zeros, wave, lane);
            b.load_end(t, left, q.zeros, wave, lane);
        }
    };
    // (behind the loop the compiler moves all of c about if it may)
    auto pin = [&](int j) {
#pragma unroll
        for (int i = 0; i < IM; ++i) {
            if constexpr (BM == 256)
                asm volatile("" : "+a"(c[i][j]));
            else
                asm volatile("" : "+v"(c[i][j]));
        }
    };
    // Half KS of a step: its matrix instructions, one after the other, and between them, where the matrix pipe is busy
    // anyway, the reads of the other half (of this step, or of the next one behind `turn`) in the first half of them, and
    // in half 1 the loads at pa and pb into the other buffer. The fences keep that order.
    auto half = [&](auto ks, const char* pa, const char* pb) {
        constexpr int KS = decltype(ks)::value, SLOTS = IM * IN, READS = IM + IN;
        static_assert(LOADS < SLOTS, "the last slot has no load");
        const uint32_t da = a.dst ^ TA::BYTES, db = b.dst ^ TB::BYTES;
        auto slot = [&](auto at) {
            constexpr int S = decltype(at)::value, i = S / IN, j = S % IN;
            constexpr int l = (S * LOADS + SLOTS - 1) / SLOTS;   // the load whose slot this is, if any
            if constexpr (KS == 1 && l < LOADS && l * SLOTS / LOADS == S) {
                if constexpr (l < TA::LOADS)
                    mfma_load<T, BM == 256, l * 1024>(fa[KS][i], fb[KS][j], c[i][j], pa, a.off[l], da);
                else
                    mfma_load<T, BM == 256, (l - TA::LOADS) * 1024>(fa[KS][i], fb[KS][j], c[i][j], pb, b.off[l - TA::LOADS], db);
            } else {
                mfma<T, BM == 256, KS == 1 && S == SLOTS - 1>(fa[KS][i], fb[KS][j], c[i][j]);
            }
#pragma unroll
            for (int r = 0; r < READS; ++r)
                if (r * SLOTS / (2 * READS) == S) {
                    if (r < IN)
                        fb[1 - KS][r] = b.read(r, 1 - KS);
                    else
                        fa[1 - KS][r - IN] = a.read(r - IN, 1 - KS);
                }
            __builtin_amdgcn_sched_barrier(0);
        };
        each(std::make_integer_sequence<int, SLOTS>{}, slot);
    };
    // Step t. Behind the last step an old buffer is read once more, for nothing, and behind the last two step 1 is loaded
    // again (the zeros, where there is only step 0), so that the loop has no branches.
    auto step = [&](int t) {
        half(std::integral_constant<int, 0>{}, nullptr, nullptr);
        // this wavefront has read the step and its loads of the next one have arrived; then everybody's
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        a.turn();
        b.turn();
        const int k = t + 2 < steps ? t + 1 : 0;
        half(std::integral_constant<int, 1>{}, a.base + k * a.step, b.base + k * b.step);
    };
    load_first();
    if (steps > 1) {
#pragma unroll
        for (int i = 0; i < TA::LOADS; ++i) a.load(0, TA::BYTES, i);
#pragma unroll
        for (int i = 0; i < TB::LOADS; ++i) b.load(0, TB::BYTES, i);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS) : "memory");
    } else {
        // there is no whole step that the loop could load again
        a.stay(q.zeros);
        b.stay(q.zeros);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    asm volatile("s_barrier" ::: "memory");
    // what the epilogue needs, so that it is not fetched behind the loop
    ProductArgs end;
    auto keep = [](auto& to, auto from) {
        to = from;
        asm volatile("" : "+s"(to));
    };
    float alpha = 0.0f;
    keep(end.M, q.M), keep(end.N, q.N);
    if constexpr (EPILOGUE == LOGITS) {
        keep(end.target, q.target), keep(end.zt, q.zt), keep(end.stat, q.stat);
        keep(end.segs, q.segs), keep(end.p, q.p), keep(end.ldp, q.ldp);
    } else {
        keep(end.C, q.C), keep(end.ldc, q.ldc), keep(end.vector, q.vector);
        keep(end.acc, q.acc), keep(end.ldacc, q.ldacc), keep(end.add, q.add);
        keep(alpha, *(const __attribute__((address_space(4))) float*)q.alpha);   // (by a scalar load)
    }
    // (scalar loads that are still under way would make the compiler wait for all LDS reads in every turn)
    __builtin_amdgcn_s_waitcnt(0xc07f);
#pragma unroll
    for (int j = 0; j < IN; ++j) fb[0][j] = b.read(j, 0);
#pragma unroll
    for (int i = 0; i < IM; ++i) fa[0][i] = a.read(i, 0);
    for (int t = 0; t < steps; ++t) step(t);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // no load into LDS outlives the workgroup

    // lane: row n = lo of C, elements m = 4 hi + 0..3 of each subtile (16 hi + 0..15 of four subtiles where SPREAD)
    if constexpr (EPILOGUE == LOGITS) {
        const long first = m0 + wm + 16 * hi;   // of the lane's columns; each group of four subtiles is 64 on
        const int inside = (int)(end.M - first < 2 * WM ? end.M - first : 2 * WM);   // of them before the vocabulary's end
        const bool whole = m0 + wm + WM <= end.M;
        T* to = (T*)end.p + (n0 + wn + lo) * end.ldp + first;
        long t[IN];   // (here, because loads between the stores would wait for those)
#pragma unroll
        for (int j = 0; j < IN; ++j) {
            const long n = n0 + wn + 16 * j + lo;
            t[j] = end.target[n < end.N ? n : end.N - 1];
        }
#pragma unroll
        for (int j = 0; j < IN; ++j) {
            const long n = n0 + wn + 16 * j + lo;
            const bool on = n < end.N;
            pin(j);
            float z[4 * IM];
#pragma unroll
            for (int i = 0; i < 4 * IM; ++i) {   // column 64 (i / 16) + i % 16
                z[i] = c[i / 4][j][i & 3];
                asm volatile("" : "+v"(z[i]));   // (read once from the accumulation registers)
            }
            if (!whole) {
#pragma unroll
                for (int i = 0; i < 4 * IM; ++i) z[i] = 64 * (i >> 4) + (i & 15) < inside ? z[i] : -INFINITY;
            }
            auto largest = [&] {   // (passes NaN by: the sum has it)
                float m = -INFINITY;
#pragma unroll
                for (int i = 0; i < 4 * IM; i += 2) m = max3(m, z[i], z[i + 1]);
                // (fmaxf, not the asm of max3: the compiler has to see what a permlane reads, which needs a wait behind it)
                return reduce_rows(fmaxf(m, z[0]), [](float a, float b) { return fmaxf(a, b); });
            };
            float m = largest();
            // The target's logit stands alone: k_finish adds its exponential to a maximum and a sum of the others, so that
            // what they leave of a sure prediction's loss is not lost beside it.
            const long target = on ? t[j] - first : -1;
            const int at = target >= 0 && target < inside ? (int)target : -1;
            const bool here = at >= 0 && at < 64 * (IM / 4) && (at & 63) < 16;
            if (__builtin_expect(__ballot(here) != 0, 0)) {
                float zt = 0.0f;
#pragma unroll
                for (int i = 0; i < 4 * IM; ++i) {
                    const bool is = at == 64 * (i >> 4) + (i & 15);
                    zt = is ? z[i] : zt;
                    z[i] = is ? -INFINITY : z[i];
                }
                if (here) end.zt[n] = zt;
                m = largest();
            }
            const Base base = base_of(m);
            if (__builtin_expect(__ballot(!within(m)) != 0, 0)) {
#pragma unroll
                for (int i = 0; i < 4 * IM; ++i) z[i] -= base.sub;
            }
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 4 * IM; ++i) z[i] = __builtin_amdgcn_exp2f(fmaf(z[i], LOG2E, -base.top));
#pragma unroll
            for (int i = 0; i < 4 * IM; ++i) sum += z[i];
            if (end.p != nullptr && on) {
#pragma unroll
                for (int g = 0; g < IM / 4; ++g) {
                    x8 e[2];
#pragma unroll
                    for (int i = 0; i < 16; ++i) e[i >> 3][i & 7] = (T)z[16 * g + i];
                    if (whole || m0 + wm + 64 * g < end.ldp) {   // (rows of p are whole 64s)
                        *(x8*)(to + 64 * g) = e[0];
                        *(x8*)(to + 64 * g + 8) = e[1];
                    }
                }
            }
            to += 16 * end.ldp;
            sum = reduce_rows(sum, [](float a, float b) { return a + b; });
            if (hi == 0 && on && m0 + wm < end.M) end.stat[n * end.segs + (m0 + wm) / WM] = make_float2(m, sum);
        }
    } else if (end.acc != nullptr) {
        float* to = end.acc + (split * end.N + n0 + wn + lo) * end.ldacc + m0 + wm + 4 * hi;
#pragma unroll
        for (int j = 0; j < IN; ++j, to += 16 * end.ldacc) {
            pin(j);
#pragma unroll
            for (int i = 0; i < IM; ++i) {
                if (n0 + wn + 16 * j + lo >= end.N || m0 + wm + 16 * i + 4 * hi >= end.M) continue;
                f32x4 v = c[i][j];
                if (end.add) v += *(f32x4*)(to + 16 * i);
                *(f32x4*)(to + 16 * i) = v;
            }
        }
    } else {
        T* to = (T*)end.C + (n0 + wn + lo) * end.ldc + m0 + wm;
        if (end.vector && m0 + BM <= end.M) {
            // Two subtiles side by side: the lanes of odd hi get the second one's elements of the lane below and give
            // theirs of the first, so that a lane has 8 neighbouring elements and four lanes 64 bytes of a row.
            to += 16 * (hi & 1) + 8 * (hi >> 1);
#pragma unroll
            for (int j = 0; j < IN; ++j, to += 16 * end.ldc) {
                const bool on = n0 + wn + 16 * j + lo < end.N;
                pin(j);
#pragma unroll
                for (int i = 0; i < IM; i += 2) {
                    typedef T x4 __attribute__((ext_vector_type(4)));
                    x4 e[2];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        e[0][r] = (T)(c[i][j][r] * alpha);
                        e[1][r] = (T)(c[i + 1][j][r] * alpha);
                    }
                    const uint2 u = __builtin_bit_cast(uint2, e[0]), v = __builtin_bit_cast(uint2, e[1]);
                    const auto x = __builtin_amdgcn_permlane16_swap(u.x, v.x, false, false);
                    const auto y = __builtin_amdgcn_permlane16_swap(u.y, v.y, false, false);
                    if (on) *(uint4*)(to + 16 * i) = make_uint4(x[0], y[0], x[1], y[1]);
                }
            }
        } else {
            const int left = (int)(end.M - m0 - wm < 4 * BM ? end.M - m0 - wm : 4 * BM) - 4 * hi;   // elements of the row
            to += 4 * hi;
#pragma unroll
            for (int j = 0; j < IN; ++j, to += 16 * end.ldc) {
                pin(j);
                if (n0 + wn + 16 * j + lo >= end.N) continue;
#pragma unroll
                for (int i = 0; i < IM; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (16 * i + r < left) to[16 * i + r] = (T)(c[i][j][r] * alpha);
            }
        }
    }
}

// The logits of few tokens (16 NB at most): bound by one read of W, which goes straight into registers, at any
// alignment. A workgroup has FEW_ROWS columns of the vocabulary; its four wavefronts share the hidden size, 32 k of every
// 128 each, and put their parts together in LDS, so that there are many loads under way (a wavefront's next four steps)
// and many wavefronts. Statistics and exponentials as in the other kernel, for FEW_ROWS columns together.
// With few tokens a single rounding of G shows in a whole gradient (no other tokens' average it away), and rows of the
// products' tiles are free: so p and G have two rows a token, the rounded values and behind all of those what was
// rounded off, and the gradients see 16 bits of them (bf16) or 21.
// 1 x 1024 x 32000: 13 us for 65 MB; the tiles above take 15, and unaligned rows would have to be copied for them.
constexpr int FEW_ROWS = 32, FEW_TOKENS = 32;
template <typename T, int NB>
__global__ __launch_bounds__(256) void k_few(const ProductArgs q) {
    typedef typename Vec<T>::x8 x8;
    constexpr int MA = FEW_ROWS / 16, AHEAD = 4;
    __shared__ float part[4][16 * NB][FEW_ROWS + 1];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, lo = lane & 15, hi = lane >> 4;
    const long m0 = (long)FEW_ROWS * blockIdx.x;
    const T *a[MA], *b[NB];
#pragma unroll
    for (int i = 0; i < MA; ++i) {
        const long row = m0 + 16 * i + lo;
        a[i] = (const T*)q.A + (row < q.M ? row : q.M - 1) * q.lda;
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const long row = 16 * j + lo;
        b[j] = (const T*)q.B + (row < q.N ? row : q.N - 1) * q.ldb;
    }
    f32x4 c[MA][NB] = {};
    auto step = [&](long k, x8(&fa)[MA], x8(&fb)[NB]) {
#pragma unroll
        for (int i = 0; i < MA; ++i) fa[i] = __builtin_bit_cast(x8, *(const Pack8<T>*)(a[i] + k));
#pragma unroll
        for (int j = 0; j < NB; ++j) fb[j] = __builtin_bit_cast(x8, *(const Pack8<T>*)(b[j] + k));
    };
    auto multiply = [&](const x8(&fa)[MA], const x8(&fb)[NB], f32x4(&d)[MA][NB]) {
#pragma unroll
        for (int i = 0; i < MA; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                if constexpr (std::is_same<T, bf16>::value)
                    d[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[i], fb[j], d[i][j], 0, 0, 0);
                else
                    d[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa[i], fb[j], d[i][j], 0, 0, 0);
            }
    };
    const long whole = q.K / 32;   // steps of 32 k without an end
    long s = wave;
    for (; s + 4 * (AHEAD - 1) < whole; s += 4 * AHEAD) {
        x8 fa[AHEAD][MA], fb[AHEAD][NB];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) step(32 * (s + 4 * u) + 8 * hi, fa[u], fb[u]);
        // a sum of its own for these 512 k: a long chain of additions would round at the whole sum's size
        f32x4 d[MA][NB] = {};
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) multiply(fa[u], fb[u], d);
#pragma unroll
        for (int i = 0; i < MA; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) c[i][j] += d[i][j];
    }
    for (; 32 * s < q.K; s += 4) {
        x8 fa[MA], fb[NB];
        const long k = 32 * s + 8 * hi;
        if (s < whole) {
            step(k, fa, fb);
        } else {
            const int n = q.K - k >= 8 ? 8 : q.K > k ? (int)(q.K - k) : 0;
#pragma unroll
            for (int r = 0; r < 8; ++r) {
#pragma unroll
                for (int i = 0; i < MA; ++i) fa[i][r] = r < n ? a[i][k + r] : (T)0.0f;
#pragma unroll
                for (int j = 0; j < NB; ++j) fb[j][r] = r < n ? b[j][k + r] : (T)0.0f;
            }
        }
        multiply(fa, fb, c);
    }
#pragma unroll
    for (int i = 0; i < MA; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) part[wave][16 * j + lo][16 * i + 4 * hi + r] = c[i][j][r];
    __syncthreads();
    // a token's columns belong to 8 lanes, four each
    for (int n = threadIdx.x >> 3; n < 16 * NB; n += 32) {
        const int col = 4 * (threadIdx.x & 7);
        const long v = m0 + col;
        const bool on = n < q.N;
        const long tgt = on ? q.target[n] : -1;
        float z[4], m = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            z[r] = (part[0][n][col + r] + part[1][n][col + r]) + (part[2][n][col + r] + part[3][n][col + r]);
            if (v + r == tgt && v + r < q.M) q.zt[n] = z[r];   // it stands alone, as in the other kernel
            if (v + r >= q.M || v + r == tgt) z[r] = -INFINITY;
            m = fmaxf(m, z[r]);
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        const Base base = base_of(m);
        typedef T x4 __attribute__((ext_vector_type(4)));
        x4 e, rest;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float x = __builtin_amdgcn_exp2f(fmaf(z[r] - base.sub, LOG2E, -base.top));
            sum += x;
            e[r] = (T)x;
            rest[r] = (T)(x - (float)e[r]);
        }
        sum = reduce_lanes<8, Sum>(sum);
        if (!on) continue;
        if (q.p != nullptr && v < q.ldp) {
            *(x4*)((T*)q.p + n * q.ldp + v) = e;
            *(x4*)((T*)q.p + (q.N + n) * q.ldp + v) = rest;
        }
        if ((threadIdx.x & 7) == 0) q.stat[n * q.segs + blockIdx.x] = make_float2(m, sum);
    }
}

struct Scalars {
    uint32_t zeros[4];
    float alpha;    // what dx and dW are multiplied by
    float per;      // what the sum of the losses is multiplied by
    float w_scale;  // G holds the weights times this (a power of 2: the largest weight to [1, 2))
};

// the sum (or mean) of the tokens' losses by one workgroup, in a fixed order
__device__ __forceinline__ void total(const float* loss, long N, const Scalars* scal, float* out) {
    __shared__ double slot[4];
    double sum = 0.0;
    long i = threadIdx.x;
    for (; i + 7 * 256 < N; i += 8 * 256) {   // (eight loads together)
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = loss[i + 256 * k];
#pragma unroll
        for (int k = 0; k < 8; ++k) sum += (double)v[k];
    }
    for (; i < N; i += 256) sum += (double)loss[i];
    sum = reduce_threads<256, Sum>(sum, slot);
    if (threadIdx.x == 0) *out = (float)(sum * (double)scal->per);
}
__global__ __launch_bounds__(256) void k_total(const float* loss, long N, const Scalars* scal, float* out) {
    total(loss, N, scal, out);
}

// C = alpha times the sum of the splits' parts, in their order, of `rows` rows each; two: of twice as many, the second
// half added to the first. Where `loss` is given, one workgroup more than JOINERS has the N tokens' total.
constexpr unsigned JOINERS = 2048;
template <typename T>
__global__ __launch_bounds__(256) void k_join(const float* acc, int splits, bool two, long rows, long M, long Mp, void* C,
                                              const Scalars* scal, const float* loss, long N, float* out) {
    if (blockIdx.x == JOINERS) return total(loss, N, scal, out);
    const long n = rows * Mp / 4;
    const int parts = two ? 2 * splits : splits;
    const float a = scal->alpha;
    for (long i = blockIdx.x * 256l + threadIdx.x; i < n; i += 256l * JOINERS) {
        f32x4 v = ((const f32x4*)acc)[i];
        int s = 1;
        for (; s + 8 <= parts; s += 8) {   // (their loads together)
            f32x4 u[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) u[k] = ((const f32x4*)acc)[(s + k) * n + i];
#pragma unroll
            for (int k = 0; k < 8; ++k) v += u[k];
        }
        for (; s < parts; ++s) v += ((const f32x4*)acc)[s * n + i];
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
    long rest;                   // elements from a row of p to the one with what was rounded off, or 0
};

// one token a blockIdx.x: lse from the segments' statistics, the loss, and p -> G in the columns of blockIdx.y.
// Bound by memory where there are gradients: 8192 x 128000, read and written, in 910 us (4.6 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void k_finish(const FinishArgs q) {
    __shared__ float slot[4];
    const long i = blockIdx.x;
    const float2* stat = q.stat + i * q.segs;
    float m = -INFINITY;
    for (long s = threadIdx.x; s < q.segs; s += 256) m = nan_max(m, stat[s].x);
    m = reduce_threads<256, NanMax>(m, slot);
    const long t = q.target[i];
    const float w = weight_of(t, q.ignore, q.V, q.row_weight, i);
    const bool column = t >= 0 && t < q.V, in = column && t != q.ignore;
    const float zt = column ? q.zt[i] : -INFINITY;
    // The segments have all but the target. Relative to the larger of their maximum and the target's logit (NaN if either is;
    // segments without a logit above -inf add exp(-inf) times their sum, 0 or NaN):
    const float most = nan_max(m, zt), top = most == -INFINITY ? 0.0f : most;
    float rest = 0.0f;
    for (long s = threadIdx.x; s < q.segs; s += 256)
        rest += stat[s].y * __builtin_amdgcn_exp2f(fmaf(stat[s].x - top, LOG2E, -off_of(stat[s].x)));
    rest = reduce_threads<256, Sum>(rest, slot);
    // log of the sum of all exponentials: of 1 + rest where the target is the largest; of at least 1 otherwise
    const float far = zt - top, l = log1pf(rest + expm1f(far));
    const float d = in ? l - far : w;   // the token's loss (or 0, or NaN)
    if (blockIdx.y == 0 && threadIdx.x == 0) {
        q.loss[i] = w == 0.0f ? 0.0f : w * d;
        if (q.lse != nullptr) q.lse[i] = top + l;
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
            if (q.rest) {
                float r[8];
                load8(p + q.rest + v, 8, r);
#pragma unroll
                for (int k = 0; k < 8; ++k) e[k] += r[k];
            }
            const float seg = stat[v < q.V ? v >> q.seg : 0].x;
            const float s = v < q.V ? f * __builtin_amdgcn_exp2f(fmaf((seg - top) - l, LOG2E, -off_of(seg))) : 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] = v + k < q.V ? e[k] * s : 0.0f;
            if (in && t >= v && t < v + 8) {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (t == v + k) e[k] = f * expm1f(-d);
            }
        }
        store8(p + v, 8, e);
        if (q.rest) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float r = e[k] - (float)(T)e[k];
                e[k] = r == r ? r : 0.0f;   // (infinite or NaN: the first row has it)
            }
            store8(p + q.rest + v, 8, e);
        }
    }
}

// rows of H elements to rows of Hp (the next multiple of 8), the rest 0: operands whose rows do not start on 16 bytes.
// `times` the same rows, one lot after the other.
template <typename T>
__global__ __launch_bounds__(256) void k_pad(const T* src, long ld, long rows, int times, long H, long Hp, T* dst) {
    const long pieces = Hp / 8;
    for (long i = blockIdx.x * 256l + threadIdx.x; i < times * rows * pieces; i += 256l * gridDim.x) {
        const long row = i / pieces, at = 8 * (i - row * pieces);
        float v[8];
        load8(src + row % rows * ld + at, H - at >= 8 ? 8 : (int)(H - at), v);
        store8(dst + row * Hp + at, 8, v);
    }
}

constexpr long MAX_N = (1l << 31) - 1, MAX_HV = 1l << 22;   // counted in int; 256 rows stay within 32-bit byte offsets

long up(long v, long to) { return (v + to - 1) / to * to; }
long over(long v, long by) { return (v + by - 1) / by; }

// the workgroup tiles: 256 x 256, 128 x 128 and 128 (m) x 64 (n)
enum { BIG, MID, NARROW };
constexpr int TILE_M[] = {256, 128, 128}, TILE_N[] = {256, 128, 64};
constexpr int SLOTS[] = {256, 512, 768};        // workgroups the device holds at once
constexpr double STEP_US[] = {1.6, 1.0, 0.95};  // 64 k of a full device, at the clock that it keeps under this load
constexpr double ALONE_US[] = {1.6, 0.6, 0.5};  // and with one workgroup a compute unit
constexpr double ENDS_US[][3] = {{9.5, 5.0, 4.0}, {8.7, 3.8, 3.5}};   // a workgroup's first loads and its epilogue: logits, others

struct Shape {
    int kind;
    long m_tiles, n_tiles;
    int splits;
    long split_k;
};

// Microseconds of C [N][M] over K in tiles of `kind`, in `splits` parts of K. Measured, in us, for 256 / 128 / 64-wide
// tiles: logits of 512 x 768 x 32000 30 / 33 / 40, of 128 x 1024 x 32000 29 / 18 / 16, of 2000 x 2048 x 50257 410 / 465 /
// 537, of 4000 x 1024 x 50257 425 / 484 / 550; dW of the same 38 / 34 / 40, 24 / 24 / 27, 370 / 428 / 531, 385 / 419 / 529; dx
// and the sum of its parts, of 512 x 768 x 32000 in 16 parts 50 + 6 / 33 + 6 / 34 + 6, in 8 80 + 5 / 44 + 5 / 39 + 5, of
// 2000 x 2048 x 50257 in 4 parts 357 + 13 / 430 + 14 / 580 + 14.
double time_of(int epilogue, int kind, long M, long N, long K, long splits) {
    const double tiles = (double)(over(M, TILE_M[kind]) * over(N, TILE_N[kind]) * splits);
    // workgroups beside each other on the compute units that have most; where there is one, nothing fills its gaps
    const double most = SLOTS[kind] / 256, beside = tiles >= SLOTS[kind] ? most : ceil(tiles / 256);
    const double step = beside <= 1 ? ALONE_US[kind] : ALONE_US[kind] + (STEP_US[kind] - ALONE_US[kind]) * (beside - 1) / (most - 1);
    const double ends = ENDS_US[epilogue][kind] + (tiles <= 256 ? 3.0 : 0.0);
    // the last round of the largest starts as workgroups end, one after the other; tiles that share a compute unit fill
    // each other's gaps
    double rounds = tiles / SLOTS[kind];
    rounds = rounds <= 1.0 ? 1.0 : kind == BIG ? 0.5 * (rounds + ceil(rounds)) : rounds;
    const double join = splits > 1 ? 3.0 + 1e-6 * (double)(M * N * splits) : 0.0;
    return rounds * (step * (double)over(over(K, 64), splits) + ends) + join;
}

// rows of fp32 sums that dx over several parts of K may take
long split_rows(long tokens) {
    const long most = 2 * tokens > 16384 ? 2 * tokens : 16384;
    const long rows = tokens <= FEW_TOKENS ? 128 * tokens : tokens <= 2 * FEW_TOKENS ? 128 * FEW_TOKENS : 64 * tokens;
    return rows < most ? rows : most;
}

// the fastest by time_of, in at most `most` parts of K
Shape shape_of(int epilogue, long M, long N, long K, long most) {
    Shape best = {};
    double least = 1e300;
    for (int kind = BIG; kind <= NARROW; ++kind)
        for (long splits = 1; splits <= most && (splits == 1 || over(K, 64) >= 4 * splits); ++splits) {
            const double t = time_of(epilogue, kind, M, N, K, splits);
            if (t < least * 0.98) {
                least = t;
                best = {kind, over(M, TILE_M[kind]), over(N, TILE_N[kind]), (int)splits, 64 * over(over(K, 64), splits)};
            }
        }
    return best;
}

// How many rows of C [N][M] to leave to the largest tiles, so that those come out in whole rounds over the device, where
// `all` has them: the rest takes smaller tiles in a launch of its own. dW of 4000 x 1024 x 50257 are 788 tiles, 20 more than
// three rounds: 350 + 50 us so, 421 in one launch.
long rows_of_rounds(const Shape& all, long M, long N, long K) {
    const long tiles = all.m_tiles * all.n_tiles, rows = TILE_N[BIG] * (tiles / SLOTS[BIG] * SLOTS[BIG] / all.m_tiles);
    if (all.kind != BIG || all.splits > 1 || rows == 0 || rows >= N) return N;
    const Shape rest = shape_of(OUT, M, N - rows, K, 1);
    return time_of(OUT, BIG, M, rows, K, 1) + time_of(OUT, rest.kind, M, N - rows, K, 1) < time_of(OUT, BIG, M, N, K, 1) ? rows : N;
}

// Where things lie in the workspace, for `tokens` tokens at a time. It does not shrink with more tokens, so that what fits for
// some fits for fewer. The sums of dx's parts come last: there are as many parts as the rest of the workspace holds.
struct Layout {
    long scal, loss, zt, stat, p, dw_acc, x, w, dx_acc, bytes;
    long rows, segs, ldp, Hp;    // (rows of p)
    int seg;                     // columns that share a maximum, 2^seg
    bool few;                    // the logits by k_few, p and G in two rows a token
    Shape logits;                // of a full piece of the tokens
};
Layout layout_of(long N, long H, long V, int grads, bool pad, long tokens) {
    Layout l;
    l.logits = shape_of(LOGITS, V, tokens, H, 1);
    l.few = tokens <= FEW_TOKENS;
    l.rows = l.few ? 2 * tokens : tokens;
    l.seg = l.few ? 5 : l.logits.kind == BIG ? 7 : 6;
    l.segs = over(V, 1l << l.seg);
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
    const long most = l.few || tokens > 2 * FEW_TOKENS ? l.rows : 2 * FEW_TOKENS;   // (not below what fewer tokens need)
    l.stat = take(8 * (l.few ? tokens * over(V, FEW_ROWS) : most * over(V, 64)));
    l.p = take(grads ? 2 * most * l.ldp : 0);
    l.dw_acc = take((grads & 2) && tokens < N ? 4 * l.Hp * V : 0);
    l.x = take(pad ? 2 * most * l.Hp : (grads & 2) ? 2 * (l.few ? l.rows : 2 * FEW_TOKENS) * l.Hp : 0);
    l.w = take(pad ? 2 * V * l.Hp : 0);
    l.dx_acc = take((grads & 1) ? 4 * (l.few ? l.rows : 2 * FEW_TOKENS) * l.Hp : 0);
    l.bytes = at;
    return l;
}

// dx of a full piece of the tokens, with sums in `bytes` bytes where there are several parts or few tokens
Shape dx_of(const Layout& l, long H, long V, long tokens, long bytes) {
    const long most = l.rows > 0 ? std::min(split_rows(tokens) / l.rows, bytes / (4 * l.rows * l.Hp)) : 1;
    return shape_of(OUT, H, l.rows, V, most > 1 ? most : 1);
}

// A launch has fewer than 2^32 threads: 256 for each of k_finish's tokens, and for each tile of the logits.
constexpr long MAX_TOKENS = 1l << 23, MAX_TILES = 1l << 24;

// most tokens at a time within `most` bytes: all, or a multiple of 256 (at least 256)
long tokens_of(long N, long H, long V, int grads, bool pad, long most) {
    auto fit = [&](long tokens, long bytes) {
        if (tokens > MAX_TOKENS) return false;
        const Layout l = layout_of(N, H, V, grads, pad, tokens);
        return l.bytes <= bytes && l.logits.m_tiles * l.logits.n_tiles < MAX_TILES;
    };
    if (N <= 256 || fit(N, most)) return N;
    long lo = 1, hi = over(N, 256);   // in units of 256: lo is taken, hi is too many
    while (hi - lo > 1) {
        const long mid = (lo + hi) / 2;
        if (fit(256 * mid, most))
            lo = mid;
        else
            hi = mid;
    }
    // the pieces alike; or all at once after all, where the pieces' sums of dW take more
    const long pieces = over(N, 256 * lo), even = std::min(up(over(N, pieces), 256), 256 * lo);
    return fit(N, layout_of(N, H, V, grads, pad, even).bytes) ? N : even;
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
        k_product<T, A_ROWS, B_ROWS, EPILOGUE, 256, 256, 128, 128><<<grid, 256, 0, st>>>(q);
    else if (s.kind == MID)
        k_product<T, A_ROWS, B_ROWS, EPILOGUE, 128, 128, 64, 64><<<grid, 256, 0, st>>>(q);
    else
        k_product<T, A_ROWS, B_ROWS, EPILOGUE, 128, 64, 64, 32><<<grid, 256, 0, st>>>(q);
}

template <typename T>
int enqueue(const Call& c, char* ws, long bytes, long tokens, hipStream_t st) {
    const int grads = (c.dx != nullptr ? 1 : 0) | (c.dw != nullptr ? 2 : 0);
    const Layout l = layout_of(c.N, c.H, c.V, grads, c.pad, tokens);
    const Shape dx = grads & 1 ? dx_of(l, c.H, c.V, tokens, bytes - l.dx_acc) : Shape{};
    Scalars* scal = (Scalars*)(ws + l.scal);
    float* loss = c.reduced ? (float*)(ws + l.loss) : c.loss;
    const T *x = (const T*)c.x, *w = (const T*)c.w;
    const long ldx = c.ldx;
    long ldw = c.ldw;
    // (each token's loss alone needs no scale, and zeros only where the hidden size is no multiple of a step)
    if (grads || c.reduced || (!l.few && l.Hp % BK != 0))
        k_prepare<<<1, 1024, 0, st>>>(c.target, c.N, c.ignore, c.mean, c.row_weight, c.grad_scale, g_scale<T>(), scal);
    auto pad_grid = [&](long rows) { return (unsigned)(over(rows * l.Hp / 8, 256) < 4096 ? over(rows * l.Hp / 8, 256) : 4096); };
    if (c.pad) {
        k_pad<T><<<pad_grid(c.V), 256, 0, st>>>(w, ldw, c.V, 1, c.H, l.Hp, (T*)(ws + l.w));
        w = (const T*)(ws + l.w);
        ldw = l.Hp;
    }
    ProductArgs base = {};
    base.zeros = scal->zeros;
    base.ldp = l.ldp, base.segs = l.segs;
    base.ldc = c.H, base.ldacc = l.Hp;
    base.alpha = &scal->alpha;
    bool totalled = false;
    // no tokens: dW is a product over nothing
    for (long at = 0; at < c.N || (at == 0 && c.dw != nullptr); at += tokens > 0 ? tokens : 1) {
        const long n = c.N - at < tokens ? c.N - at : tokens;
        const T* xs = x + at * ldx;   // this piece's tokens
        long ldxs = ldx;
        const bool two = l.few && n > 0;   // rows a token in p, and x twice for dW
        if (n > 0 && (c.pad || (two && c.dw != nullptr))) {
            const int times = two && c.dw != nullptr ? 2 : 1;
            k_pad<T><<<pad_grid(times * n), 256, 0, st>>>(xs, ldx, n, times, c.H, l.Hp, (T*)(ws + l.x));
            xs = (const T*)(ws + l.x);
            ldxs = l.Hp;
        }
        if (n > 0) {
            ProductArgs q = base;
            q.M = c.V, q.N = n, q.K = c.pad ? l.Hp : c.H;
            q.A = w, q.lda = ldw;
            q.B = xs, q.ldb = ldxs;
            q.target = c.target + at;
            q.zt = (float*)(ws + l.zt);
            q.stat = (float2*)(ws + l.stat);
            q.p = grads ? ws + l.p : nullptr;
            Shape s = l.logits;
            s.n_tiles = over(n, TILE_N[s.kind]);
            if (!l.few)
                product<T, true, true, LOGITS>(s, q, st);
            else if (n <= 16)
                k_few<T, 1><<<(unsigned)l.segs, 256, 0, st>>>(q);
            else
                k_few<T, 2><<<(unsigned)l.segs, 256, 0, st>>>(q);
            FinishArgs f = {c.V, l.segs, l.ldp, c.ignore, l.seg, c.target + at,
                            c.row_weight == nullptr ? nullptr : c.row_weight + at, q.zt, q.stat, q.p, loss + at,
                            c.lse == nullptr ? nullptr : c.lse + at, scal, two ? n * l.ldp : 0};
            const long split = grads ? (n >= 2048 ? 1 : 2048 / n) : 1, most = over(l.ldp, 2048);
            k_finish<T><<<dim3((unsigned)n, (unsigned)(split < most ? split : most)), 256, 0, st>>>(f);
        }
        if (c.dx != nullptr && n > 0) {
            ProductArgs d = base;
            d.M = c.H, d.N = two ? 2 * n : n, d.K = c.V;
            d.A = w, d.lda = ldw;
            d.B = ws + l.p, d.ldb = l.ldp;
            T* C = (T*)c.dx + at * c.H;
            d.C = C;
            d.vector = c.H % 8 == 0 && (uintptr_t)C % 16 == 0;
            d.acc = two || dx.splits > 1 ? (float*)(ws + l.dx_acc) : nullptr;
            Shape s = dx;
            s.n_tiles = over(d.N, TILE_N[s.kind]);
            product<T, false, true, OUT>(s, d, st);
            if (d.acc != nullptr) {
                const bool last = c.reduced && at + n == c.N;   // the losses are all there
                k_join<T><<<JOINERS + last, 256, 0, st>>>(d.acc, s.splits, two, n, c.H, l.Hp, C, scal, loss, c.N, c.loss);
                totalled |= last;
            }
        }
        if (c.dw != nullptr) {
            ProductArgs d = base;
            d.M = c.H, d.N = c.V, d.K = two ? 2 * n : n;
            d.A = xs, d.lda = ldxs;
            d.B = ws + l.p, d.ldb = l.ldp;
            d.C = c.dw;
            d.vector = c.H % 8 == 0 && (uintptr_t)c.dw % 16 == 0;
            d.acc = tokens < c.N ? (float*)(ws + l.dw_acc) : nullptr;
            d.add = at > 0;
            Shape s = shape_of(OUT, c.H, c.V, d.K, 1);
            const long rows = rows_of_rounds(s, c.H, c.V, d.K);
            if (rows < c.V) {
                d.N = rows, s.n_tiles = rows / TILE_N[BIG];
                product<T, false, false, OUT>(s, d, st);
                d.N = c.V - rows;
                d.B = (const T*)d.B + rows;
                d.C = (T*)d.C + rows * c.H;
                if (d.acc != nullptr) d.acc += rows * l.Hp;
                s = shape_of(OUT, c.H, d.N, d.K, 1);
            }
            product<T, false, false, OUT>(s, d, st);
            if (d.acc != nullptr && at + n == c.N)
                k_join<T><<<JOINERS, 256, 0, st>>>((const float*)(ws + l.dw_acc), 1, false, c.V, c.H, l.Hp, c.dw, scal, nullptr, 0, nullptr);
        }
    }
    if (c.reduced && !totalled) k_total<<<1, 256, 0, st>>>(loss, c.N, scal, c.loss);
    return launched("linear_cross_entropy");
}

}  // namespace

extern "C" {

long spanqr_linear_cross_entropy_workspace(int type, long N, long H, long V, int grads, long most_bytes) {
    const int rc = check_sizes(type, N, H, V);
    if (rc != SPANQR_OK) return rc;
    const bool pad = ((grads & 4) || H % 8 != 0) && ((grads & 3) || N > FEW_TOKENS);
    const long tokens = tokens_of(N, H, V, grads & 3, pad, most_bytes);
    const Layout l = layout_of(N, H, V, grads & 3, pad, tokens);
    if (!(grads & 1)) return l.bytes;
    // (what is beyond most_bytes anyway has room for all parts of dx)
    const Shape dx = dx_of(l, H, V, tokens, N > 256 && l.bytes <= most_bytes ? most_bytes - l.dx_acc : LONG_MAX);
    return std::max(l.bytes, dx.splits > 1 ? l.dx_acc + 4 * dx.splits * l.rows * l.Hp : 0);
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
    // (few tokens' losses take any alignment)
    const bool pad = needs_pad(x, N > 1 ? ldx : 0, w, V > 1 ? ldw : 0, H) && (grads || N > FEW_TOKENS);
    const long tokens = tokens_of(N, H, V, grads, pad, workspace_bytes), need = layout_of(N, H, V, grads, pad, tokens).bytes;
    if (need > workspace_bytes) return error(SPANQR_EINVAL, "linear_cross_entropy: the workspace needs %ld bytes", need);
    const Call c = {reduction == SPANQR_REDUCE_MEAN, reduced, pad, N, H, V, x, w, ldx, ldw, target, ignore_index,
                    row_weight, grad_scale, loss, lse, dx, dw};
    hipStream_t st = (hipStream_t)stream;
    return type == SPANQR_BF16 ? enqueue<bf16>(c, (char*)workspace, workspace_bytes, tokens, st)
                               : enqueue<fp16>(c, (char*)workspace, workspace_bytes, tokens, st);
}

}  // extern "C"
