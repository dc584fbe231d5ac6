// attention.hip -- softmax attention with heads that share keys and values, for padded batches and packed sequences, and its
// gradient, which makes the probabilities again.
//
//   S = c Q K^T,  lse_i = log sum_j exp S_ij,  P_ij = exp(S_ij - lse_i),  O = P V
//   D_i = sum_d dO_id O_id,  dP = dO V^T,  dS = P (dP - D),  dV = P^T dO,  dK = c dS^T Q,  dQ = c dS K
//   query i of a sequence stands at p = i + Lk - Lq; causal: j <= p, with a window w also j > p - w; a query that sees no key
//   has O = 0, lse = -inf and no gradient
//
// A group of G heads shares a key head; its queries are taken as Lq G rows (row m is query m / G of head m % G), so that
// what is read of K and V serves the whole group, one token of a group fills a tile, and the gradient of shared heads is a sum
// over rows like any other: no atomics, the same bits in every call.
//
// All products are of 32 x 32 x 16 matrix instructions, arranged so that what one leaves in registers is what the next one
// takes: a lane of S^T (K's rows against Q's) has 16 keys of one query, which are the softmax's to reduce (one lane swap joins
// the two halves) and, rounded to 16 bits, the second operand of O^T = V^T P^T, the sum over keys going in the order in
// which they lie in the registers. V^T comes from LDS by the transposing read in that order. The gradient of K and V
// holds its keys by lanes and streams Q and dO; that of Q holds queries and streams K and V. P is rounded to 16 bits before
// the product with V or dO, and dS before those with K and Q; all sums are fp32.
//
// fp16 holds nothing below 2^-24, and little below 2^-14. So there P goes into its products times a power of two that keeps it
// below 2^15, and dS times one that a bound on it allows: |dP_ij - D_i| <= 2 |dO_i| |V_j|, the lane's own norm and the other
// side's largest. The powers go into the exponent, and the results are divided by them. bf16 has fp32's exponents.
#include <limits.h>
#include <math.h>

#include <type_traits>

#include "elements.h"
#include "host.h"

using namespace spanqr_dev;
using spanqr_host::error;
using spanqr_host::launched;

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 fp16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN2 = 0.69314718055994530942f;
constexpr int TILE = 64;     // rows of a tile in LDS
constexpr int WAVES = 4;
constexpr int BLOCK = 32 * WAVES;   // rows that a workgroup holds, a wavefront 32

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

// c + a b, 32 x 32 x 16: lane l has row l % 32 of a and column l % 32 of b, k = 8 (l / 32) + 0..7 of both, and of c the column
// l % 32, register i being row 8 (i / 4) + 4 (l / 32) + i % 4
__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma(fp16x8 a, fp16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// log2 of what P is multiplied by: over a base that may be 2^8 too small in the forward pass, and at most 1 in the backward pass
template <typename T>
constexpr float raised(bool forward) { return std::is_same<T, fp16>::value ? (forward ? 7.0f : 14.0f) : 0.0f; }
// log2 of what dS, at most 2 sqrt(a b), may be multiplied by to stay within 2^14
__device__ __forceinline__ float room(float a, float b) {
    const float most = 2.0f * sqrtf(a) * sqrtf(b);
    if (!(most > 0.0f && most < INFINITY)) return 0.0f;
    const float e = 13.0f - floorf(__builtin_amdgcn_logf(most));
    return fminf(fmaxf(e, -60.0f), 60.0f);
}
// x, or 0 where it is not finite (a row of such numbers gives such gradients, whatever the others are multiplied by)
__device__ __forceinline__ float finite(float x) { return x < INFINITY ? x : 0.0f; }
// the largest of n partial maxima, in every lane
__device__ __forceinline__ float largest(const float* p, int n, int lane) {
    float m = 0.0f;
    for (int i = lane; i < n; i += 64) m = fmaxf(m, p[i]);
    return reduce_lanes<64, NanMax>(m);
}

// registers 8 s to 8 s + 7 in 16 bits
template <typename T>
__device__ __forceinline__ typename Vec<T>::x8 half_of(const f32x16& v, int s) {
    typename Vec<T>::x8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (T)v[8 * s + i];
    return r;
}

// of the lane with the same l % 32 in the other half, and this one's
template <typename OP>
__device__ __forceinline__ float both_halves(float v, OP op) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a = r[0], b = r[1];   // (a bit_cast of a vector's element takes the first one)
    return op(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}

// N products whose first operands come from LDS, AHEAD of them under way: the compiler left to itself reads each operand right
// before its product and waits for it. between(i): what else goes behind product i.
template <int N, int AHEAD, typename X8, typename READ, typename PRODUCT, typename BETWEEN>
__device__ __forceinline__ void stream(X8 (&f)[AHEAD], READ read, PRODUCT product, BETWEEN between) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        product(i, f[i % AHEAD]);
        if (i + AHEAD < N) f[i % AHEAD] = read(i + AHEAD);
        between(i);
        __builtin_amdgcn_sched_barrier(0);
    }
}
template <int AHEAD, typename X8, typename READ>
__device__ __forceinline__ void read_ahead(X8 (&f)[AHEAD], READ read) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) f[i] = read(i);
    __builtin_amdgcn_sched_barrier(0);
}

// One of q, k, v, out, dout: elements between batches, rows and heads; 16-byte alignment, neighbouring elements of a head.
struct Heads {
    const void* p;
    long batch, row, head;
};

struct Shape {
    int B, Hk, G, D;              // sequences, key heads, heads a key head, elements a head
    long Tq, Tk;                  // rows of all sequences; of each one where nothing is packed
    const int *q_starts, *k_starts;   // packed: B + 1 each, ascending; or null
    const int* k_lens;            // not packed: B numbers of keys, or null: Tk
    int causal, window;           // window 0: none
    float scale2;                 // c log2 e
};

// where a sequence's rows lie: the first one among all, and how many
struct Seq {
    long q0, k0;
    int lq, lk;
};
__device__ __forceinline__ void span(const int* starts, int b, long T, long& at, int& n) {
    const long a = starts[b] < 0 ? 0 : starts[b] > T ? T : starts[b];
    const long e = starts[b + 1] < a ? a : starts[b + 1] > T ? T : starts[b + 1];
    at = a;
    n = (int)(e - a);
}
__device__ __forceinline__ Seq seq_of(const Shape& s, int b) {
    Seq r;
    if (s.q_starts != nullptr) {
        span(s.q_starts, b, s.Tq, r.q0, r.lq);
        span(s.k_starts, b, s.Tk, r.k0, r.lk);
    } else {
        const int n = s.k_lens != nullptr ? s.k_lens[b] : (int)s.Tk;
        r = {b * s.Tq, b * s.Tk, (int)s.Tq, n < 0 ? 0 : n < s.Tk ? n : (int)s.Tk};
    }
    return r;
}
// the first row of a sequence and a head
template <typename T>
__device__ __forceinline__ const char* head_of(const Heads& h, bool packed, int b, long row0, int head) {
    return (const char*)h.p + (long)sizeof(T) * ((packed ? row0 * h.row : b * h.batch) + head * h.head);
}

// what a load reads outside a matrix: elements past D, rows past the end
__device__ const uint32_t __attribute__((aligned(16))) nothing[4] = {0, 0, 0, 0};
__device__ const float no_row[2] = {INFINITY, 0.0f};   // lse and -D of a row past the end

// 16 bytes (4) a lane to LDS at `lds` + 16 lane (4 lane), asynchronously: counted by vmcnt, which `arrived` waits for
__device__ __forceinline__ void load_lds(const char* base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory");
}
__device__ __forceinline__ void load_lds(const void* at, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(at) : "memory");
}
__device__ __forceinline__ void load_lds4(const void* at, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(at) : "memory");
}
// this wavefront's loads are there and its reads are done; then everybody's
__device__ __forceinline__ void arrived() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Tiles of 64 rows of PITCH elements (64 or 128) in LDS, of which DP (D rounded up to a multiple of 32) are used, and the way
// there and into registers. The 16-byte chunk c of a row lies at c ^ swizzle(row): LDS serves lanes 0-3, 12-15, 20-27 of each 32 together and
// then the others, 256 bytes at a time, and for reads of rows (16 rows, the same chunk) as for transposing reads (4 rows,
// 64 bytes of each) those fill the 256 bytes exactly.
template <int PITCH>
__device__ __forceinline__ int swizzle(int row) {
    return PITCH == 128 ? (row & 3) << 2 | (row >> 2 & 3) : (row >> 1 & 1) << 2 | (row >> 2 & 3);
}

template <typename T, int PITCH>
struct Reader {
    typedef typename Vec<T>::x8 x8;
    static constexpr int ROW = 2 * PITCH;            // bytes
    static constexpr int BYTES = TILE * ROW;
    uint32_t rows, cols[2];                       // a lane's places in a tile, or with the tile's address added
    __device__ __forceinline__ explicit Reader(int lane) {
        const int r = lane & 31, h = lane >> 5, lo = lane & 15, g = lane >> 4 & 1;
        rows = r * ROW + ((swizzle<PITCH>(r) ^ h) << 4);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int k = 8 * j + 4 * h + (lo >> 2);
            cols[j] = k * ROW + (((2 * g + (lo >> 1 & 1)) ^ swizzle<PITCH>(k)) << 4) + 8 * (lo & 1);
        }
    }
    __device__ __forceinline__ Reader(const Reader& r, uint32_t tile) : rows(r.rows + tile), cols{r.cols[0] + tile, r.cols[1] + tile} {}
    __device__ __forceinline__ void move(int by) {
        rows += by;
        cols[0] += by;
        cols[1] += by;
    }
    // makes the compiler form the places below again behind this point: kept, they take the registers of two results
    __device__ __forceinline__ void fresh() { asm volatile("" : "+v"(rows), "+v"(cols[0]), "+v"(cols[1])); }
    // rows 32 t + lane % 32, elements 16 ks + 8 (lane / 32) + 0..7, of the tile `off` bytes on
    __device__ __forceinline__ x8 row(int off, int t, int ks) const {
        return *(__attribute__((address_space(3))) const x8*)(uintptr_t)((rows ^ 32 * ks) + off + t * 32 * ROW);
    }
    // element 32 dt + lane % 32 of the rows 16 s + 4 (lane / 32) + 0..3 and those + 8: the order of a result's registers
    __device__ __forceinline__ x8 col(int off, int s, int dt) const {
        typedef __attribute__((address_space(3))) s16x4 lds_s4;
        const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)((cols[0] ^ 64 * dt) + off + s * 16 * ROW));
        const s16x4 w = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)((cols[1] ^ 64 * dt) + off + s * 16 * ROW));
        return __builtin_bit_cast(x8, __builtin_shufflevector(v, w, 0, 1, 2, 3, 4, 5, 6, 7));
    }
};

// Loads of tiles of rows m of one sequence and key head, m / G being the row in memory and m % G the head. A tile has
// rows_of_tile(G) rows, whole rows in memory, so that a lane's places are the same in every tile, and a tile inside the matrix
// is loaded from a base that moves. (What it has behind D is the row's last 16 bytes again: the other operand is 0 there, or
// the result is not used. What it has behind its rows is the last one again: there the probabilities are 0.) At the matrix's end
// every lane finds its own, and reads zeros past it. Groups of which a tile's whole rows would leave too much empty are
// taken 64 rows a tile, each lane finding its own always.
// KEPT: the places stay in registers; otherwise in LDS, a lane's own words.
__device__ __forceinline__ int rows_of_tile(int G) {
    const int n = G <= TILE ? TILE / G * G : 0;
    return n >= TILE - 8 ? n : TILE;
}
template <typename T, int PITCH, bool KEPT>
struct Loader {
    static constexpr int CHUNKS = PITCH / 8, LOADS = TILE * CHUNKS / 64 / WAVES;
    static constexpr int TABLE = KEPT ? 0 : 16 * 64 * WAVES;   // bytes of LDS
    static_assert(KEPT || LOADS == 4, "");
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) u32x4 lds_u4;
    const char* base;
    long row, head;       // bytes
    int G, rows, last;    // last: the row's last chunk
    uint32_t table, off[KEPT ? LOADS : 1];
    __device__ __forceinline__ static int row_of(int i, int wave, int lane) { return (wave * LOADS + i) * (64 / CHUNKS) + lane / CHUNKS; }
    __device__ __forceinline__ int chunk_of(int r, int lane) const {
        const int c = lane % CHUNKS ^ swizzle<PITCH>(r);
        return c < last ? c : last;
    }
    __device__ __forceinline__ Loader(const char* base, const Heads& h, int G, int D, int wave, int lane, uint32_t table = 0)
        : base(base), row((long)sizeof(T) * h.row), head((long)sizeof(T) * h.head), G(G), rows(rows_of_tile(G)), last(D / 8 - 1), table(table) {
        u32x4 all;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int r = row_of(i, wave, lane), m = r < rows ? r : rows - 1;
            // (strides stay below 2^25 bytes)
            const uint32_t at = (uint32_t)(m / G) * (uint32_t)row + (uint32_t)(m % G) * (uint32_t)head + 16 * chunk_of(r, lane);
            if constexpr (KEPT)
                off[i] = at;
            else
                all[i] = at;
        }
        if constexpr (!KEPT) *(lds_u4*)(uintptr_t)(table + 16 * threadIdx.x) = all;
    }
    // the tile of rows from m0 (a multiple of `rows`) on, of M, into LDS
    __device__ __forceinline__ void load(int m0, int M, uint32_t lds, int wave, int lane) const {
        const uint32_t to = lds + wave * LOADS * 1024;
        if (rows % G == 0 && m0 + rows <= M) {
            const char* from = base + (m0 / G) * row;
            if constexpr (KEPT) {
#pragma unroll
                for (int i = 0; i < LOADS; ++i) load_lds(from, off[i], to + i * 1024);
            } else {
                uint32_t mine = threadIdx.x;
                asm volatile("" : "+v"(mine));
                const u32x4 all = *(const lds_u4*)(uintptr_t)(table + 16 * mine);
#pragma unroll
                for (int i = 0; i < LOADS; ++i) load_lds(from, all[i], to + i * 1024);
            }
        } else {
            asm volatile("" : "+v"(lane));   // (formed here: hoisted, the places would fill the registers)
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int r = row_of(i, wave, lane), m = m0 + r, q = m / G;
                const void* from = m < M ? (const void*)(base + q * row + (m - q * G) * head + 16 * chunk_of(r, lane)) : (const void*)nothing;
                load_lds(from, to + i * 1024);
            }
        }
    }
};

// the second operand straight from memory: a lane's row at p (or nothing)
template <typename T, int DP>
__device__ __forceinline__ void load_row(const char* p, bool on, int D, int lane, typename Vec<T>::x8 (&f)[DP / 16]) {
    asm volatile("" : "+v"(lane));   // (nothing of it is kept for the next block)
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
        const int d = 16 * ks + 8 * (lane >> 5);
        const char* from = on && d < D ? p + sizeof(T) * d : (const char*)nothing;
        f[ks] = *(const typename Vec<T>::x8*)from;
    }
}

// a result's column (a row of D elements in memory at p) times f, 16 bytes a lane
template <typename T, int DP>
__device__ __forceinline__ void store_row(T* p, bool on, int D, int lane, const f32x16 (&c)[DP / 32], float f) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    typedef T x4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
            x4 v, w;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = (T)(c[dt][4 * q + i] * f);
                w[i] = (T)(c[dt][4 * q + 4 + i] * f);
            }
            const u32x2 a = __builtin_bit_cast(u32x2, v), b = __builtin_bit_cast(u32x2, w);
            // the lower half of the lanes gets both halves' elements 8 q + 0..7, the upper one 8 q + 8..15
            const auto lo = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false);
            const auto hi = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
            const int d = 32 * dt + 8 * q + 8 * (lane >> 5);
            const u32x4 out = {lo[0], hi[0], lo[1], hi[1]};
            if (on && d < D) *(u32x4*)(p + d) = out;
        }
}

// Zeros in rows [0, from) and [to, T) of `width` elements (a multiple of 8), by workgroups `me` of `all`; rest (or null): -inf
// for each of the `per` heads of such a row
template <typename T>
__device__ void outside(T* p, float* rest, long from, long to, long rows, long width, int per, long me, long all) {
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const long t = me * 256 + threadIdx.x, step = all * 256;
    for (long i = t; i < from * width / 8; i += step) ((uint4*)p)[i] = zero;
    for (long i = to * width / 8 + t; i < rows * width / 8; i += step) ((uint4*)p)[i] = zero;
    if (rest == nullptr) return;
    for (long i = t; i < from * per; i += step) rest[i] = -INFINITY;
    for (long i = to * per + t; i < rows * per; i += step) rest[i] = -INFINITY;
}
__device__ __forceinline__ long clip_start(int s, long T) { return s < 0 ? 0 : s > T ? T : s; }

// What workgroups are dealt out by: tiles of EACH rows (of `per` a row in memory), a sequence's and key head's `n` each, a
// workgroup taking every step-th of them where it has more. Or, where `work` is not 0, one list a key head for all sequences of a packed
// call: slot start_b per / EACH + b + t is tile t of sequence b. A sequence's slots lie behind each other and are as many as its
// tiles, or one more, so that `work` slots are enough whatever the lengths are, which the host does not know. Behind them come
// the workgroups for the rows of no sequence.
struct Tiles {
    int n, work, step;
};
struct Place {
    int b, hk, split, first;   // b: B for rows of no sequence (first: of how many, see `others`), -1 for a slot without a tile
};
template <int EACH>
__device__ __forceinline__ int slot_of(const int* starts, int b, long T, int per) {
    return (int)((uint64_t)(clip_start(starts[b], T) * per) / EACH) + b;
}
// The last sequence whose slots begin at `slot` or before, or -1: each wavefront's lanes look at 64 of them at a time. (Whatever
// the starts hold, it ends, and looks at B + 1 of them.)
template <int EACH>
__device__ __forceinline__ int sequence_of(const int* starts, int B, long T, int per, int slot) {
    const int lane = threadIdx.x & 63;
    int b = 0, n = B + 1;
    while (true) {
        const int step = (n + 63) / 64, at = b + lane * step;
        const int k = __popcll(__ballot(lane * step < n && slot_of<EACH>(starts, at < B ? at : B, T, per) <= slot));
        if (k == 0) return -1;
        b += (k - 1) * step;
        n -= (k - 1) * step;
        if (step == 1) return b < B ? b : -1;
        n = n < step ? n : step;
    }
}
// LAST: a sequence's last tiles first. extra: with workgroups for the rows of no sequence
template <int EACH, bool LAST>
__device__ __forceinline__ Place place_of(const Shape& s, const Tiles& t, const int* starts, long T, int per, bool extra) {
    const int many = t.work == 0 ? (s.B + (extra ? 1 : 0)) * s.Hk : s.Hk;
    const int which = blockIdx.x % many, turn = blockIdx.x / many, split = turn / t.n;
    const int first = LAST ? t.n - 1 - turn % t.n : turn % t.n;
    if (t.work == 0) return {which / s.Hk, which % s.Hk, split, first};
    if (first >= t.work) return {s.B, which, split, first - t.work};
    const int b = sequence_of<EACH>(starts, s.B, T, per, first), tile = b < 0 ? -1 : first - slot_of<EACH>(starts, b, T, per);
    return {tile < 0 ? -1 : b, which, split, tile};   // (below 0: starts that do not ascend)
}
__device__ __forceinline__ int others(const Tiles& t) { return t.work == 0 ? t.n : t.n - t.work; }
// the maxima that the workgroups of a sequence and key head leave, one for each slot: the first one's place and how many
__device__ __forceinline__ int maxima_of(const Shape& s, const Tiles& t, int b, int hk, long row0, int rows, int& n) {
    if (t.work == 0) {
        n = t.n;
        return (b * s.Hk + hk) * t.n;
    }
    const int from = (int)((uint64_t)row0 / BLOCK);
    n = (int)((uint64_t)(row0 + rows) / BLOCK) + 1 - from;
    return hk * t.work + from + b;
}

struct ForwardArgs {
    Shape s;
    Heads q, k, v;
    void* out;            // [rows of all][heads][D]
    float* lse;           // [rows of all][heads], or null
    Tiles tiles;
    int splits;
    float* part;          // splits > 1: [split][rows of all x heads][D] sums, and behind them float2 (base, sum) for each
    long rows;            // rows of all x heads
};

// A workgroup has 128 rows, a wavefront 32 of them in registers (a lane one query), and goes over the keys in tiles of 64 in
// two LDS buffers. The softmax's base moves only where a tile's maximum is more than 2^8 above it: sums and products are
// relative to it anyway, and 64 multiplications a tile and lane are left out. Bound by the matrix pipe and the softmax's vector
// instructions (5 for each product of 32 cycles at 128 wide heads, 13 at 64), at a clock that falls with what both draw: 16384 x 40 x 128 on 8 heads, causal,
// bf16 2.7 ms, 1.0 PFLOP/s; 16 x 1024 x 12 x 64 46 us; 4 x 1999 x 16 x 80 with every key seen 113. A token of 40 heads against 8191 keys
// of 8 is bound by latency, 10.1 us for 34 MB, and 3.5 for k_join.
template <typename T, int DP>
__global__ __launch_bounds__(64 * WAVES, 2) void k_forward(const ForwardArgs a) {
    typedef typename Vec<T>::x8 x8;
    constexpr int PITCH = DP <= 64 ? 64 : 128;
    typedef Reader<T, PITCH> R;
    constexpr int AHEAD = 4;
    __shared__ __attribute__((aligned(1024))) char smem[4 * R::BYTES];
    const Shape& s = a.s;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
    const bool packed = s.q_starts != nullptr;
    // all heads' longest rows of keys first; neighbouring heads go round the XCDs, so that a head's tiles meet in one L2
    const Place place = place_of<BLOCK, true>(s, a.tiles, s.q_starts, s.Tq, s.G, packed && a.splits == 1);
    const int b = place.b, hk = place.hk, split = place.split, first = place.first;
    if (b < 0) return;
    if (b == s.B) {
        outside((T*)a.out, a.lse, clip_start(s.q_starts[0], s.Tq), clip_start(s.q_starts[s.B], s.Tq), s.Tq, (long)s.Hk * s.G * s.D,
                s.Hk * s.G, first * s.Hk + hk, others(a.tiles) * s.Hk);
        return;
    }
    const Seq seq = seq_of(s, b);
    const int M = seq.lq * s.G, ahead = seq.lk - seq.lq;   // query i stands at i + ahead
    const R read(lane);
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_char*)smem;
    const Loader<T, PITCH, true> K(head_of<T>(a.k, packed, b, seq.k0, hk), a.k, 1, s.D, wave, lane);
    const Loader<T, PITCH, true> V(head_of<T>(a.v, packed, b, seq.k0, hk), a.v, 1, s.D, wave, lane);
    const char* q = head_of<T>(a.q, packed, b, seq.q0, hk * s.G);
    // keys of this split
    const int chunk = a.splits == 1 ? seq.lk : ((seq.lk + a.splits - 1) / a.splits + TILE - 1) / TILE * TILE;
    const int k_from = split * chunk < seq.lk ? split * chunk : seq.lk, k_to = k_from + chunk < seq.lk ? k_from + chunk : seq.lk;

    for (int tile = first; (long)tile * BLOCK < M; tile += a.tiles.step) {
        const int m0 = tile * BLOCK, w0 = m0 + 32 * wave, m = w0 + (lane & 31);
        const int i = (m < M ? m : M - 1) / s.G, g = m - i * s.G;
        const bool on = m < M;
        x8 fq[DP / 16];
        load_row<T, DP>(q + (long)sizeof(T) * (i * a.q.row + g * a.q.head), on, s.D, lane, fq);
        // the keys [lo, hi) that this lane's query sees, this wavefront's queries see, and the workgroup's
        const int hi = s.causal ? (i + ahead + 1 < k_to ? i + ahead + 1 : k_to) : k_to;
        const int lo = s.window && i + ahead - s.window + 1 > k_from ? i + ahead - s.window + 1 : k_from;
        const int i_first = w0 / s.G, i_last = ((w0 + 31 < M ? w0 + 31 : M - 1)) / s.G;
        const int all_hi = s.causal ? (i_first + ahead + 1 < k_to ? i_first + ahead + 1 : k_to) : k_to;
        const int any_hi = w0 >= M ? 0 : s.causal ? (i_last + ahead + 1 < k_to ? i_last + ahead + 1 : k_to) : k_to;
        const int any_lo = s.window && i_first + ahead - s.window + 1 > k_from ? i_first + ahead - s.window + 1 : k_from;
        const int all_lo = s.window && i_last + ahead - s.window + 1 > k_from ? i_last + ahead - s.window + 1 : k_from;
        const int block_last = (m0 + BLOCK < M ? m0 + BLOCK : M) - 1;
        const int to = k_from == k_to ? 0 : s.causal ? (block_last / s.G + ahead + 1 < k_to ? block_last / s.G + ahead + 1 : k_to) : k_to;
        int from = s.window && m0 / s.G + ahead - s.window + 1 > k_from ? m0 / s.G + ahead - s.window + 1 : k_from;
        from &= ~(TILE - 1);

        f32x16 o[DP / 32] = {};
        float base = -INFINITY, sum = 0.0f;   // the base is in units of log2
        // both buffers at once: a split of a long cache has two tiles, and one memory latency then
        for (int i = 0; i < 2; ++i)
            if (from + i * TILE < to) {
                K.load(from + i * TILE, seq.lk, lds + 2 * i * R::BYTES, wave, lane);
                V.load(from + i * TILE, seq.lk, lds + 2 * i * R::BYTES + R::BYTES, wave, lane);
            }
        uint32_t now = lds;
        for (int n0 = from; n0 < to; n0 += TILE, now = 2 * lds + 2 * R::BYTES - now) {
            arrived();
            if (n0 != from && n0 + TILE < to) {
                const uint32_t other = 2 * lds + 2 * R::BYTES - now;
                K.load(n0 + TILE, seq.lk, other, wave, lane);
                V.load(n0 + TILE, seq.lk, other + R::BYTES, wave, lane);
            }
            if (n0 >= any_hi || n0 + TILE <= any_lo) continue;
            const R in(read, now);
            f32x16 z[2] = {};
            x8 f[AHEAD];
            const auto keys = [&](int i) { return in.row(0, i % 2, i / 2); };
            read_ahead(f, keys);
            stream<DP / 8>(f, keys, [&](int i, x8 k) { z[i % 2] = mfma(k, fq[i / 2], z[i % 2]); }, [](int) {});
            // (the first of the values are read while the softmax goes on)
            const auto values = [&](int i) { return in.col(R::BYTES, i / (DP / 32), i % (DP / 32)); };
            read_ahead(f, values);
            if (n0 + TILE > all_hi || n0 < all_lo) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int j = n0 + 32 * t + 8 * (r / 4) + 4 * h + r % 4;
                        z[t][r] = j >= lo && j < hi ? z[t][r] : -INFINITY;
                    }
            }
            float top = z[0][0];
#pragma unroll
            for (int r = 1; r < 32; ++r) top = fmaxf(top, z[r / 16][r % 16]);
            top = both_halves(top, [](float x, float y) { return fmaxf(x, y); }) * s.scale2;
            if (__any(top > base + 8.0f)) {
                const float next = fmaxf(base, top), down = next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(base - next);
                base = next;
                sum *= down;
#pragma unroll
                for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[dt][r] *= down;
            }
            const float off = base == -INFINITY ? 0.0f : base - raised<T>(true);
            // a tile's sum first: one chain over all keys is off by up to 2^-24 for every other key, and by as much to one side
            // where probabilities are alike (2^-11 for 65536 keys)
            float add = 0.0f;
            const auto exps = [&](int t, int from, int to) {
#pragma unroll
                for (int r = from; r < to; ++r) {
                    z[t][r] = __builtin_amdgcn_exp2f(fmaf(z[t][r], s.scale2, -off));
                    add += z[t][r];
                }
            };
            exps(0, 0, 16);
            x8 p[2] = {half_of<T>(z[0], 0), half_of<T>(z[0], 1)};
            __builtin_amdgcn_sched_barrier(0);
            constexpr int DT = DP / 32, EACH = (16 + 2 * DT - 1) / (2 * DT);
            stream<4 * DT>(f, values, [&](int i, x8 v) { o[i % DT] = mfma(v, p[i / DT % 2], o[i % DT]); }, [&](int i) {
                if (i < 2 * DT) exps(1, EACH * i, EACH * (i + 1) < 16 ? EACH * (i + 1) : 16);
                if (i == 2 * DT - 1) p[0] = half_of<T>(z[1], 0), p[1] = half_of<T>(z[1], 1);
            });
            sum += add;
        }
        sum = both_halves(sum, [](float x, float y) { return x + y; });
        base -= raised<T>(true);
        const long at = (seq.q0 + i) * (s.Hk * s.G) + hk * s.G + g;
        if (a.splits == 1) {
            store_row<T, DP>((T*)a.out + at * s.D, on, s.D, lane, o, sum == 0.0f ? 0.0f : 1.0f / sum);
            if (on && h == 0 && a.lse != nullptr) a.lse[at] = sum == 0.0f ? -INFINITY : (base + __builtin_amdgcn_logf(sum)) * LN2;
        } else if (on) {
            float* part = a.part + (split * a.rows + at) * s.D;
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) {
                    const int d = 32 * dt + 8 * q4 + 4 * h;
                    if (d < s.D) *(float4*)(part + d) = make_float4(o[dt][4 * q4], o[dt][4 * q4 + 1], o[dt][4 * q4 + 2], o[dt][4 * q4 + 3]);
                }
            if (h == 0) ((float2*)(a.part + a.splits * a.rows * s.D))[split * a.rows + at] = make_float2(base, sum);
        }
        arrived();   // (nobody reads the buffers any more)
    }
}

// The splits' sums joined: a workgroup a row, each wavefront every fourth split, a lane two elements (D <= 128); in a fixed
// order. A wavefront has JOINED splits' loads under way at once and joins them as the forward pass joins tiles, so that 64
// splits cost one memory latency (a pass for the maximum first: 5.2 us instead of 4.0 for 40 rows of 63 splits).
template <typename T, int JOINED>
__global__ __launch_bounds__(64 * WAVES) void k_join(const ForwardArgs a) {
    __shared__ float add[WAVES][4][64];
    const Shape& s = a.s;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, heads = s.Hk * s.G;
    const float2* stat = (const float2*)(a.part + a.splits * a.rows * s.D);
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        bool in = true;
        if (s.q_starts != nullptr) {
            const long row = r / heads;
            in = row >= clip_start(s.q_starts[0], s.Tq) && row < clip_start(s.q_starts[s.B], s.Tq);
        }
        float top = -INFINITY, sum = 0.0f, x = 0.0f, y = 0.0f;
        const long d = r * s.D + (2 * lane < s.D ? 2 * lane : 0);
        for (int i0 = wave; in && i0 < a.splits; i0 += JOINED * WAVES) {
            float2 v[JOINED], p[JOINED];
#pragma unroll
            for (int j = 0; j < JOINED; ++j) {
                const long i = i0 + j * WAVES < a.splits ? i0 + j * WAVES : i0;
                v[j] = stat[i * a.rows + r];
                p[j] = *(const float2*)(a.part + i * a.rows * s.D + d);
            }
            float next = top;
#pragma unroll
            for (int j = 0; j < JOINED; ++j)
                if (i0 + j * WAVES < a.splits) next = fmaxf(next, v[j].x);
            const float down = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - next);
            sum *= down, x *= down, y *= down;
            top = next;
#pragma unroll
            for (int j = 0; j < JOINED; ++j) {
                // (no visible key: zeros)
                const float w = i0 + j * WAVES >= a.splits || v[j].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(v[j].x - top);
                sum = fmaf(v[j].y, w, sum);
                x = fmaf(p[j].x, w, x);
                y = fmaf(p[j].y, w, y);
            }
        }
        add[wave][0][lane] = top;
        add[wave][1][lane] = sum;
        add[wave][2][lane] = x;
        add[wave][3][lane] = y;
        __syncthreads();
        if (wave == 0) {
            float all = top;
#pragma unroll
            for (int w = 1; w < WAVES; ++w) all = fmaxf(all, add[w][0][lane]);
            sum = x = y = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const float t = add[w][0][lane], f = t == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(t - all);
                sum = fmaf(add[w][1][lane], f, sum);
                x = fmaf(add[w][2][lane], f, x);
                y = fmaf(add[w][3][lane], f, y);
            }
            const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
            if (2 * lane < s.D) {
                T* out = (T*)a.out + r * s.D + 2 * lane;
                out[0] = (T)(x * f);
                out[1] = (T)(y * f);
            }
            if (lane == 0 && a.lse != nullptr) a.lse[r] = sum == 0.0f ? -INFINITY : (all + __builtin_amdgcn_logf(sum)) * LN2;
        }
        __syncthreads();
    }
}

struct BackwardArgs {
    Shape s;
    Heads q, k, v, out, dout;
    const float* lse;
    void *dq, *dk, *dv;   // contiguous
    float* stat;          // [2][rows of all x heads], from k_dq: lse log2 e (inf where nothing is seen), -D
    long rows;
    Tiles q_tiles, k_tiles, kv_tiles;
    float scale;
    float *v_most, *d_most;   // fp16: the largest |V_j|^2 and |dO_i|^2 of each workgroup of k_tiles and q_tiles
    int q_splits, kv_splits;  // workgroups that share a tile, each going over a part of the other side
    float *q_part, *k_part, *v_part;   // [split][rows of all x heads][D], where there is more than one
};

// the split's share of [from, to), which it takes in steps of `step`
__device__ __forceinline__ void share(int split, int splits, int step, int& from, int& to) {
    if (splits == 1 || from >= to) return;
    const int each = ((to - from + step - 1) / step + splits - 1) / splits * step;
    const long at = from + (long)split * each;
    from = at < to ? (int)at : to;
    to = to - from > each ? from + each : to;
}

// a result's column as it is, times f, 16 bytes a lane
template <int DP>
__device__ __forceinline__ void store_part(float* p, bool on, int D, int lane, const f32x16 (&c)[DP / 32], float f) {
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int d = 32 * dt + 8 * q + 4 * (lane >> 5);
            if (on && d < D) *(float4*)(p + d) = make_float4(c[dt][4 * q] * f, c[dt][4 * q + 1] * f, c[dt][4 * q + 2] * f, c[dt][4 * q + 3] * f);
        }
}

// Sums of the splits' parts, in their order, eight elements a thread; zeros in rows of no sequence. One launch for all three.
struct Parts {
    const float* part;
    void* out;
    const int* starts;        // packed: B + 1
    long rows, width;         // of all sequences; elements of a row
    int splits;               // 1: nothing to do
};
struct PartsArgs {
    Parts of[3];
    int B;
};
template <typename T>
__global__ __launch_bounds__(256) void k_parts(const PartsArgs a) {
    const Parts& p = a.of[blockIdx.y];
    if (p.splits == 1) return;
    const long n = p.rows * p.width;
    const long begin = p.starts != nullptr ? clip_start(p.starts[0], p.rows) : 0, end = p.starts != nullptr ? clip_start(p.starts[a.B], p.rows) : p.rows;
    for (long i = 8 * (blockIdx.x * 256l + threadIdx.x); i < n; i += 8l * 256 * gridDim.x) {
        const long row = i / p.width;
        const bool in = row >= begin && row < end;
        float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int k = 0; k < p.splits; ++k) {
            const float4 x = *(const float4*)(p.part + k * n + i), y = *(const float4*)(p.part + k * n + i + 4);
            sum[0] += x.x, sum[1] += x.y, sum[2] += x.z, sum[3] += x.w, sum[4] += y.x, sum[5] += y.y, sum[6] += y.z, sum[7] += y.w;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] = in ? sum[j] : 0.0f;
        store8((T*)p.out + i, 8, sum);
    }
}

// |V_j|^2's maxima over a workgroup's rows: 16 lanes a row, eight elements a lane
template <typename T>
__global__ __launch_bounds__(64 * WAVES) void k_v_most(const BackwardArgs a) {
    __shared__ float slot[WAVES];
    const Shape& s = a.s;
    const Place place = place_of<BLOCK, false>(s, a.k_tiles, s.k_starts, s.Tk, 1, false);
    const int b = place.b, hk = place.hk, first = place.first;
    if (b < 0) return;
    const Seq seq = seq_of(s, b);
    const T* v = (const T*)head_of<T>(a.v, s.q_starts != nullptr, b, seq.k0, hk);
    const int d = 8 * (threadIdx.x & 15), here = s.D - d >= 8 ? 8 : 0;
    float most = 0.0f;
    for (int tile = first; (long)tile * BLOCK < seq.lk; tile += a.k_tiles.step)
        for (int j = tile * BLOCK + (threadIdx.x >> 4); j < (tile + 1) * BLOCK && j < seq.lk; j += 16) {
            float x[8], sum = 0.0f;
            load8(v + j * a.v.row + d, here, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fmaf(x[e], x[e], sum);
            most = fmaxf(most, finite(reduce_lanes<16, Sum>(sum)));
        }
    most = reduce_threads<64 * WAVES, NanMax>(most, slot);
    int n;
    if (threadIdx.x == 0) a.v_most[maxima_of(s, a.k_tiles, b, hk, seq.k0, seq.lk, n) + first] = most;
}

// dQ: as the forward pass, 128 rows a workgroup; a lane has one query. It has dO in registers, so it forms D first, and leaves it
// and lse as the gradients take it for the keys' kernel (a pass of its own over O and dO took 15 us of 200 at 16 x 1024 x 12 x 64).
// Without dq that is all it does. 16384 x 40 x 128 on 8 heads, causal, bf16: 3.3 ms, 1.24 PFLOP/s, the matrix pipe busy for 73 % of
// the cycles at 1.6 GHz; 16 x 1024 x 12 x 64 58 us.
template <typename T, int DP>
__global__ __launch_bounds__(64 * WAVES, 2) void k_dq(const BackwardArgs a) {
    typedef typename Vec<T>::x8 x8;
    constexpr int PITCH = DP <= 64 ? 64 : 128;
    typedef Reader<T, PITCH> R;
    constexpr int AHEAD = DP == 32 ? 2 : 4, BEHIND = DP == 32 ? 2 : 4;
    __shared__ __attribute__((aligned(1024))) char smem[4 * R::BYTES];
    const Shape& s = a.s;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
    const bool packed = s.q_starts != nullptr;
    const Place place = place_of<BLOCK, true>(s, a.q_tiles, s.q_starts, s.Tq, s.G, packed);
    const int b = place.b, hk = place.hk, split = place.split, first = place.first;
    if (b < 0) return;
    if (b == s.B) {
        if (a.dq != nullptr && a.q_splits == 1)
            outside((T*)a.dq, nullptr, clip_start(s.q_starts[0], s.Tq), clip_start(s.q_starts[s.B], s.Tq), s.Tq, (long)s.Hk * s.G * s.D, 0,
                    first * s.Hk + hk, others(a.q_tiles) * s.Hk);
        return;
    }
    const Seq seq = seq_of(s, b);
    const int M = seq.lq * s.G, ahead = seq.lk - seq.lq;
    const R read(lane);
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_char*)smem;
    const Loader<T, PITCH, true> K(head_of<T>(a.k, packed, b, seq.k0, hk), a.k, 1, s.D, wave, lane);
    const Loader<T, PITCH, true> V(head_of<T>(a.v, packed, b, seq.k0, hk), a.v, 1, s.D, wave, lane);
    const char* q = head_of<T>(a.q, packed, b, seq.q0, hk * s.G);
    const char* d_out = head_of<T>(a.dout, packed, b, seq.q0, hk * s.G);
    const char* out = head_of<T>(a.out, packed, b, seq.q0, hk * s.G);
    constexpr bool SMALL = std::is_same<T, fp16>::value;
    float v_most = 0.0f, d_most = 0.0f;
    if constexpr (SMALL) {
        int n;
        const int from = maxima_of(s, a.k_tiles, b, hk, seq.k0, seq.lk, n);
        v_most = largest(a.v_most + from, n, lane);
    }

    for (int tile = first; (long)tile * BLOCK < M; tile += a.q_tiles.step) {
        const int m0 = tile * BLOCK, w0 = m0 + 32 * wave, m = w0 + (lane & 31);
        const int i = (m < M ? m : M - 1) / s.G, g = m - i * s.G;
        const bool on = m < M;
        const long at = (seq.q0 + i) * (s.Hk * s.G) + hk * s.G + g;
        x8 fq[DP / 16], fd[DP / 16];
        load_row<T, DP>(q + (long)sizeof(T) * (i * a.q.row + g * a.q.head), on, s.D, lane, fq);
        load_row<T, DP>(d_out + (long)sizeof(T) * (i * a.dout.row + g * a.dout.head), on, s.D, lane, fd);
        float lse = INFINITY, delta = 0.0f, up = 0.0f;
        if constexpr (SMALL) {
            float sum = 0.0f;
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
                for (int e = 0; e < 8; ++e) sum = fmaf((float)fd[ks][e], (float)fd[ks][e], sum);
            sum = finite(both_halves(sum, [](float x, float y) { return x + y; }));
            d_most = fmaxf(d_most, sum);
            up = room(sum, v_most);
        }
        {
            x8 fo[DP / 16];
            load_row<T, DP>(out + (long)sizeof(T) * (i * a.out.row + g * a.out.head), on, s.D, lane, fo);
            if (on) lse = a.lse[at] == -INFINITY ? INFINITY : a.lse[at] * LOG2E;
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
                for (int e = 0; e < 8; ++e) delta = fmaf((float)fo[ks][e], (float)fd[ks][e], delta);
            delta = both_halves(delta, [](float x, float y) { return x + y; });
            if (on && h == 0 && split == 0) {
                a.stat[at] = lse - raised<T>(false);
                a.stat[a.rows + at] = -delta;
            }
        }
        if (a.dq == nullptr) continue;
        lse -= up;
        f32x16 start;   // of dP - D's sum
#pragma unroll
        for (int r = 0; r < 16; ++r) start[r] = -delta;
        const int k_to = seq.lk;
        const int hi = s.causal ? (i + ahead + 1 < k_to ? i + ahead + 1 : k_to) : k_to;
        const int lo = s.window && i + ahead - s.window + 1 > 0 ? i + ahead - s.window + 1 : 0;
        const int i_first = w0 / s.G, i_last = ((w0 + 31 < M ? w0 + 31 : M - 1)) / s.G;
        const int all_hi = s.causal ? (i_first + ahead + 1 < k_to ? i_first + ahead + 1 : k_to) : k_to;
        const int any_hi = w0 >= M ? 0 : s.causal ? (i_last + ahead + 1 < k_to ? i_last + ahead + 1 : k_to) : k_to;
        const int any_lo = s.window && i_first + ahead - s.window + 1 > 0 ? i_first + ahead - s.window + 1 : 0;
        const int all_lo = s.window && i_last + ahead - s.window + 1 > 0 ? i_last + ahead - s.window + 1 : 0;
        const int block_last = (m0 + BLOCK < M ? m0 + BLOCK : M) - 1;
        int to = s.causal ? (block_last / s.G + ahead + 1 < k_to ? block_last / s.G + ahead + 1 : k_to) : k_to;
        int from = s.window && m0 / s.G + ahead - s.window + 1 > 0 ? m0 / s.G + ahead - s.window + 1 : 0;
        from &= ~(TILE - 1);
        share(split, a.q_splits, TILE, from, to);

        f32x16 dq[DP / 32] = {};
        for (int i = 0; i < 2; ++i)
            if (from + i * TILE < to) {
                K.load(from + i * TILE, seq.lk, lds + 2 * i * R::BYTES, wave, lane);
                V.load(from + i * TILE, seq.lk, lds + 2 * i * R::BYTES + R::BYTES, wave, lane);
            }
        uint32_t now = lds;
        for (int n0 = from; n0 < to; n0 += TILE, now = 2 * lds + 2 * R::BYTES - now) {
            arrived();
            if (n0 != from && n0 + TILE < to) {
                const uint32_t other = 2 * lds + 2 * R::BYTES - now;
                K.load(n0 + TILE, seq.lk, other, wave, lane);
                V.load(n0 + TILE, seq.lk, other + R::BYTES, wave, lane);
            }
            if (n0 >= any_hi || n0 + TILE <= any_lo) continue;
            const bool masked = n0 + TILE > all_hi || n0 < all_lo;
            R in(read, now);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                in.fresh();
                f32x16 z = {}, dp = start;
                x8 f[AHEAD];
                const auto keys = [&](int i) { return in.row(0, t, i); };
                const auto values = [&](int i) { return in.row(R::BYTES, t, i); };
                read_ahead(f, keys);
                stream<DP / 16>(f, keys, [&](int i, x8 x) { z = mfma(x, fq[i], z); }, [](int) {});
                read_ahead(f, values);
                constexpr int EACH = 256 / DP;
                stream<DP / 16>(f, values, [&](int i, x8 x) { dp = mfma(x, fd[i], dp); }, [&](int i) {
#pragma unroll
                    for (int r = EACH * i; r < EACH * (i + 1) && r < 16; ++r) z[r] = __builtin_amdgcn_exp2f(fmaf(z[r], s.scale2, -lse));
                });
#pragma unroll
                for (int r = EACH * (DP / 16); r < 16; ++r) z[r] = __builtin_amdgcn_exp2f(fmaf(z[r], s.scale2, -lse));
                const auto cols = [&](int i) { return in.col(0, 2 * t + i / (DP / 32), i % (DP / 32)); };
                x8 c[BEHIND];
                read_ahead(c, cols);
#pragma unroll
                for (int r = 0; r < 16; ++r) z[r] *= dp[r];
                if (masked) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int j = n0 + 32 * t + 8 * (r / 4) + 4 * h + r % 4;
                        z[r] = j >= lo && j < hi ? z[r] : 0.0f;
                    }
                }
                const x8 ds[2] = {half_of<T>(z, 0), half_of<T>(z, 1)};
                __builtin_amdgcn_sched_barrier(0);
                stream<DP / 16>(c, cols, [&](int i, x8 x) { dq[i % (DP / 32)] = mfma(x, ds[i / (DP / 32)], dq[i % (DP / 32)]); }, [](int) {});
            }
        }
        const float times = SMALL ? a.scale * __builtin_amdgcn_exp2f(-up) : a.scale;
        if (a.q_splits == 1)
            store_row<T, DP>((T*)a.dq + at * s.D, on, s.D, lane, dq, times);
        else
            store_part<DP>(a.q_part + (split * a.rows + at) * s.D, on, s.D, lane, dq, times);
        arrived();
    }
    if (SMALL && split == 0) {
        d_most = reduce_threads<64 * WAVES, NanMax>(d_most, (float*)smem);
        int n;
        if (threadIdx.x == 0) a.d_most[maxima_of(s, a.q_tiles, b, hk, seq.q0 * s.G, M, n) + first] = d_most;
    }
}

// dK and dV: 128 keys a workgroup, a wavefront 32 of them in registers (a lane one key), over all rows of the group's
// queries that see them; or (SPLIT 2, where 128 keys would leave too few workgroups) 64 keys, two wavefronts sharing 32 and each
// taking half of every tile's rows. The rows come in tiles of 64, or as many whole queries' rows as that holds. Each product's
// first operand comes from LDS, which at 128 bytes a cycle feeds no more than the four pipes take. 16384 x 40 x 128 on 8 heads,
// causal, bf16: 5.5 ms, 0.99 PFLOP/s; 16 x 1024 x 12 x 64 72 us. Sums of dQ by the same kernel would save two of seven products, but need
// atomics, or 4 bytes of partial sums for each 128 keys and element of dQ.
template <typename T, int DP, int SPLIT>
__global__ __launch_bounds__(64 * WAVES, DP <= 64 ? 3 : 2) void k_dkv(const BackwardArgs a) {
    typedef typename Vec<T>::x8 x8;
    constexpr int PITCH = DP <= 64 ? 64 : 128;
    typedef Reader<T, PITCH> R;
    typedef Loader<T, PITCH, PITCH == 64> L;
    constexpr int AHEAD = 2, KEYS = BLOCK / SPLIT;
    constexpr int BUFFER = 2 * R::BYTES, STATS = 2 * 2 * TILE * 4 + 256;   // (and a lane's place in a tile's statistics)
    __shared__ __attribute__((aligned(1024))) char smem[2 * BUFFER + STATS + 2 * L::TABLE];
    const Shape& s = a.s;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const bool packed = s.q_starts != nullptr;
    const Place place = place_of<KEYS, false>(s, a.kv_tiles, s.k_starts, s.Tk, 1, packed);   // (the first keys are seen by most)
    const int b = place.b, hk = place.hk, split = place.split, first = place.first;
    if (b < 0) return;
    if (b == s.B) {
        if (a.kv_splits > 1) return;
        const long from = clip_start(s.k_starts[0], s.Tk), to = clip_start(s.k_starts[s.B], s.Tk), width = (long)s.Hk * s.D;
        outside((T*)a.dk, nullptr, from, to, s.Tk, width, 0, first * s.Hk + hk, others(a.kv_tiles) * s.Hk);
        outside((T*)a.dv, nullptr, from, to, s.Tk, width, 0, first * s.Hk + hk, others(a.kv_tiles) * s.Hk);
        return;
    }
    const Seq seq = seq_of(s, b);
    const int M = seq.lq * s.G, ahead = seq.lk - seq.lq;
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_char*)smem, stats = lds + 2 * BUFFER;
    const L Q(head_of<T>(a.q, packed, b, seq.q0, hk * s.G), a.q, s.G, s.D, wave, lane, stats + STATS);
    const L DO(head_of<T>(a.dout, packed, b, seq.q0, hk * s.G), a.dout, s.G, s.D, wave, lane, stats + STATS + L::TABLE);
    const int rows = Q.rows;   // of a tile
    typedef __attribute__((address_space(3))) int lds_int;
    if (wave < 2) *(lds_int*)(uintptr_t)(stats + 1024 + 4 * lane) = lane / s.G * (s.Hk * s.G) + lane % s.G;   // (both the same)
    const float* stat = a.stat + seq.q0 * (s.Hk * s.G) + hk * s.G;
    const char* k = head_of<T>(a.k, packed, b, seq.k0, hk);
    const char* v = head_of<T>(a.v, packed, b, seq.k0, hk);
    constexpr bool SMALL = std::is_same<T, fp16>::value;
    float d_most = 0.0f;
    if constexpr (SMALL) {
        int n;
        const int from = maxima_of(s, a.q_tiles, b, hk, seq.q0 * s.G, M, n);
        d_most = largest(a.d_most + from, n, lane);
    }
    const long all_keys = (packed ? s.Tk : s.B * s.Tk) * s.Hk;
    const int behind = packed ? seq.lk : (int)s.Tk;   // keys with gradients: those that lie behind k_lens have zeros
    auto load = [&](int m0, int buffer) {
        Q.load(m0, M, lds + buffer * BUFFER, wave, lane);
        DO.load(m0, M, lds + buffer * BUFFER + R::BYTES, wave, lane);
        if (wave < 2) {   // lse by one wavefront, -D by another
            int mine = lane;
            asm volatile("" : "+v"(mine));   // (nothing of it is kept)
            const int m = m0 + mine, heads = s.Hk * s.G;
            const long at = rows % s.G == 0 ? (long)(m0 / s.G) * heads + *(const lds_int*)(uintptr_t)(stats + 1024 + 4 * mine)
                                            : (long)(m / s.G) * heads + m % s.G;
            load_lds4(m < M && mine < rows ? stat + wave * a.rows + at : no_row + wave, stats + (2 * buffer + wave) * TILE * 4);
        }
    };

    for (int tile = first; (long)tile * KEYS < behind; tile += a.kv_tiles.step) {
        const int n0 = tile * KEYS, w0 = n0 + 32 * (wave % (WAVES / SPLIT)), j = w0 + (lane & 31);
        const bool on = j < seq.lk;
        x8 fk[DP / 16], fv[DP / 16];
        load_row<T, DP>(k + (long)sizeof(T) * j * a.k.row, on, s.D, lane, fk);
        load_row<T, DP>(v + (long)sizeof(T) * j * a.v.row, on, s.D, lane, fv);
        float up = 0.0f, times = 1.0f;   // dS is multiplied by 2^up, and P by 2^raised already
        if constexpr (SMALL) {
            float sum = 0.0f;
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
                for (int e = 0; e < 8; ++e) sum = fmaf((float)fv[ks][e], (float)fv[ks][e], sum);
            up = room(finite(both_halves(sum, [](float x, float y) { return x + y; })), d_most);
            times = __builtin_amdgcn_exp2f(up - raised<T>(false));
        }
        // the rows that see a key; then those that see any and all of this wavefront's keys, and the workgroup's
        auto first_row = [&](int key) {
            const long m = s.causal ? (long)(key - ahead) * s.G : 0;
            return m < 0 ? 0 : m < M ? (int)m : M;
        };
        auto end_row = [&](int key) {
            const long m = s.window ? (long)(key - ahead + s.window) * s.G : M;
            return m < 0 ? 0 : m < M ? (int)m : M;
        };
        const int last = w0 + 31 < seq.lk ? w0 + 31 : seq.lk - 1, block_last = n0 + KEYS < seq.lk ? n0 + KEYS - 1 : seq.lk - 1;
        const int any_lo = first_row(w0), any_hi = w0 < seq.lk ? end_row(last) : 0;
        const int all_lo = first_row(last), all_hi = w0 + 32 <= seq.lk ? end_row(w0) : 0;
        int from = first_row(n0) / rows * rows, to = n0 < seq.lk ? end_row(block_last) : 0;
        share(split, a.kv_splits, rows, from, to);

        f32x16 dk[DP / 32] = {}, dv[DP / 32] = {};
        if (from < to) load(from, 0);
        int buffer = 0;
        const int mine = SPLIT == 2 ? wave / 2 : 0;   // the half of a tile's rows that this wavefront takes
        R in(R(lane), lds + mine * 32 * R::ROW);
        // (threadIdx and what follows from it: formed where it is used, the registers are full)
        auto thread = [] {
            uint32_t t = threadIdx.x;
            asm volatile("" : "+v"(t));
            return t;
        };
        for (int m0 = from; m0 < to; m0 += rows, in.move(buffer ? -BUFFER : BUFFER), buffer ^= 1) {
            arrived();
            if (m0 + rows < to) load(m0 + rows, buffer ^ 1);
#pragma unroll
            for (int t = 0; t < 2 / SPLIT; ++t) {
                const int r0 = m0 + 32 * (mine + t);
                if (r0 >= any_hi || r0 + 32 <= any_lo) continue;
                in.fresh();
                const uint32_t half = (thread() >> 5 & 1) * 16 + stats + 2 * buffer * TILE * 4 + 32 * (mine + t) * 4;
                // four rows' lse or -D
                auto stat4 = [&](int which, int q4) {
                    const uint32_t at = half + (which * TILE + 8 * q4) * 4;
                    return *(__attribute__((address_space(3))) const f32x4*)(uintptr_t)at;
                };
                // dP - D: the sum starts at -D
                f32x16 z = {}, dp;
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) {
                    const f32x4 d = stat4(1, q4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) dp[4 * q4 + e] = d[e];
                }
                x8 f[AHEAD];
                const auto q_rows = [&](int i) { return in.row(0, t, i); };
                const auto do_rows = [&](int i) { return in.row(R::BYTES, t, i); };
                read_ahead(f, q_rows);
                stream<DP / 16>(f, q_rows, [&](int i, x8 x) { z = mfma(x, fk[i], z); }, [](int) {});
                read_ahead(f, do_rows);
                const auto exps = [&](int q4) {
                    const f32x4 lse = stat4(0, q4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[4 * q4 + e] = __builtin_amdgcn_exp2f(fmaf(z[4 * q4 + e], s.scale2, -lse[e]));
                };
                constexpr int EVERY = DP >= 64 ? DP / 64 : 1;   // products between four rows' exponentials
                stream<DP / 16>(f, do_rows, [&](int i, x8 x) { dp = mfma(x, fv[i], dp); }, [&](int i) {
                    if (i % EVERY == 0 && i / EVERY < 4) exps(i / EVERY);
                });
#pragma unroll
                for (int q4 = DP / 16 / EVERY; q4 < 4; ++q4) exps(q4);
                if (r0 < all_lo || r0 + 32 > all_hi) {
                    const int key = w0 + (thread() & 31), h = thread() >> 5 & 1;
                    const int lo = first_row(key), hi = key < seq.lk ? end_row(key) : 0;
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int m = r0 + 8 * (r / 4) + 4 * h + r % 4;
                        z[r] = m >= lo && m < hi ? z[r] : 0.0f;
                    }
                }
                constexpr int DT = DP / 32, EACH = (16 + 2 * DT - 1) / (2 * DT);
                const x8 p[2] = {half_of<T>(z, 0), half_of<T>(z, 1)};
                const auto do_cols = [&](int i) { return in.col(R::BYTES, 2 * t + i / DT, i % DT); };
                const auto q_cols = [&](int i) { return in.col(0, 2 * t + i / DT, i % DT); };
                read_ahead(f, do_cols);
                stream<2 * DT>(f, do_cols, [&](int i, x8 x) { dv[i % DT] = mfma(x, p[i / DT], dv[i % DT]); }, [&](int i) {
#pragma unroll
                    for (int r = EACH * i; r < EACH * (i + 1) && r < 16; ++r) dp[r] *= SMALL ? z[r] * times : z[r];
                });
                const x8 ds[2] = {half_of<T>(dp, 0), half_of<T>(dp, 1)};
                read_ahead(f, q_cols);
                stream<2 * DT>(f, q_cols, [&](int i, x8 x) { dk[i % DT] = mfma(x, ds[i / DT], dk[i % DT]); }, [](int) {});
            }
        }
        if constexpr (SPLIT == 2) {   // the other half's sums, through the tiles' memory
            constexpr int N = 16 * (DP / 32);
            typedef __attribute__((address_space(3))) float lds_float;
            lds_float* sums = (lds_float*)(uintptr_t)lds + wave % 2 * 2 * N * 64 + lane;
            arrived();
            if (mine != 0) {
#pragma unroll
                for (int r = 0; r < N; ++r) {
                    sums[64 * r] = dk[r / 16][r % 16];
                    sums[64 * (N + r)] = dv[r / 16][r % 16];
                }
            }
            arrived();
            if (mine != 0) {
                arrived();
                continue;
            }
#pragma unroll
            for (int r = 0; r < N; ++r) {
                dk[r / 16][r % 16] += sums[64 * r];
                dv[r / 16][r % 16] += sums[64 * (N + r)];
            }
        }
        const int key = w0 + (thread() & 31);
        const long at = ((seq.k0 + key) * s.Hk + hk) * s.D;
        const float k_times = SMALL ? a.scale * __builtin_amdgcn_exp2f(-up) : a.scale, v_times = SMALL ? __builtin_amdgcn_exp2f(-raised<T>(false)) : 1.0f;
        if (a.kv_splits == 1) {
            store_row<T, DP>((T*)a.dk + at, key < behind, s.D, lane, dk, k_times);
            store_row<T, DP>((T*)a.dv + at, key < behind, s.D, lane, dv, v_times);
        } else {
            const long in = split * all_keys * s.D + at;
            store_part<DP>(a.k_part + in, key < behind, s.D, lane, dk, k_times);
            store_part<DP>(a.v_part + in, key < behind, s.D, lane, dv, v_times);
        }
        arrived();
    }
}

constexpr long MAX_ROWS = 1l << 30;      // queries x group, or keys, of a sequence
constexpr long MAX_GRID = (1l << 24) - 1;
constexpr long MAX_STRIDE = 1l << 24;    // of rows, and of heads that share keys: a tile's offsets stay within 32 bits

long tiles_in(long n, long each) { return n < 1 ? 1 : (n + each - 1) / each; }

// Whether the tiles of packed sequences are one list: where those of B sequences, each as long as the longest one (or as all rows, if
// that is not known), would be more than twice as many. Forward / gradient in us with a list / without: 256 texts of up to 973 in
// 131072 rows x 40 on 8 x 128 without max_q 1620 / 4742 against 15831 / 27229, 24 of 1024 x 8 on 2 x 128 90 / 345 against 132 / 431. A
// sequence's tiles lie behind each other there, where else all sequences' longest ones go first: at 24 unlike ones whose longest is
// known, with 1.5 times the workgroups, 106 / 415 against 101 / 369.
bool as_list(bool packed, long B, long all, long longest, long each) { return packed && 2 * (all / each + B) < B * tiles_in(longest, each); }

// Tiles of `each` rows, with hints about as many as there are. (Rows that a hint too small says nothing of count too: parts are
// held for all rows.)
long count_of(bool packed, long B, long all, long longest, long each) {
    const long n = as_list(packed, B, all, longest, each) ? all / each + B : B * tiles_in(longest, each);
    return packed && n < tiles_in(all, each) ? tiles_in(all, each) : n;
}

// The tiles that workgroups are launched for. Behind a list, for `extra`, 256 workgroups for rows of no sequence. A launch takes fewer than
// 2^32 threads, 2^24 workgroups: where there are more tiles, each goes over several. n = 0: too many even so.
Tiles tiles_of(bool packed, long B, long Hk, long all, long longest, long each, long splits, bool extra) {
    const long slots = all / each + B, tail = !extra ? 0 : slots * Hk < 256 ? slots : (255 + Hk) / Hk, most = MAX_GRID / ((B + 1) * Hk * splits);
    long n = tiles_in(longest, each);
    if (as_list(packed, B, all, longest, each) && (slots + tail) * Hk * splits <= MAX_GRID) return {(int)(slots + tail), (int)slots, 1 << 24};
    n = n < most ? n : most;
    return {(int)n, 0, (int)n};
}

// Where there are few workgroups the keys are split among several, so that 512 (two for each compute unit) run, each with
// 128 keys at least; the sums are joined by a second kernel.
long splits_of(long have, long max_k) {
    if (have == 0 || have >= 256) return 1;
    const long want = (512 + have - 1) / have, most = max_k / 128;
    const long n = want < most ? want : most;
    return n < 1 ? 1 : n;
}

// The workgroups of k_dq and k_dkv that the device runs at once, by the registers that the compiler reports: three a compute unit of
// up to 64 wide heads (k_dq in bf16 takes 166, k_dkv 168), but two of k_dq in fp16 above 32 (178); two of wider heads. Both ways in us
// with three for fp16's too / two: causal 5 x 2048 x 8 x 64 192 / 170, 8 x 1024 x 10 x 64 136 / 116. Up to 32 wide in bf16 four would run
// (123): with four 5 x 2048 x 10 x 32 161 instead of 139, 1 x 1362 x 8 on 1 x 32 65 instead of 70.
long dq_at_once(int type, long D) { return 256 * (D > 64 || (type == SPANQR_FP16 && D > 32) ? 2 : 3); }
long dkv_at_once(long D) { return 256 * (D > 64 ? 2 : 3); }

// Whether the gradient of K and V takes 64 keys a workgroup: where 128 make no more than the device runs at once. Both ways in us with 128 / 64: 8 x 1024 x 8 x 128 on 4 heads
// 160 / 139, 16 x 512 x 16 x 64 on 4 116 / 98, packed 24 x 2048 x 8 x 64 on 2 357 / 294; with more of them 16 x 1024 x 12 x 64 190 / 204.
bool few_keys(long tiles, long slots) { return tiles <= slots; }

// Workgroups that share a tile of dQ's rows, or of dK's and dV's, each with four tiles of the other side at least: as many as run
// at once, or one more where a mask makes tiles uneven. Both ways in us without / with: 1 x 1362 x 8 on 1 x 64 284 / 81, causal
// 1 x 2048 x 16 on 2 x 128 480 / 199, 1 x 8192 x 2 on 1 x 64 448 / 203, 3 x 4685 x 15 on 3 x 40 814 / 676. Only where tiles make less than half
// of what runs at once 304 instead of 257 (causal 8 x 1185 x 10 on 2 x 128 fp16); one more without a mask too 201 instead of
// 177 (2 x 2277 x 3 x 128 fp16).
long grad_splits_of(long tiles, long others, long slots, int causal) {
    if (tiles >= slots) return 1;
    const long want = (causal ? slots + tiles - 1 : slots) / tiles, most = others / 4;
    const long n = want < most ? want : most;
    return n < 1 ? 1 : n;
}

struct Call {
    Shape s;
    long rows, keys;           // of all sequences, times heads
    long splits;
    bool few_keys;             // the gradient of K and V takes 64 keys a workgroup
    long q_splits, kv_splits;  // of the gradient
    Tiles tiles, q_tiles, k_tiles, kv_tiles;   // of the forward pass and the gradient
};

int check_shape(const char* what, int type, long B, long Hk, long G, long D, long Tq, long Tk, const int* q_starts,
                const int* k_starts, const int* k_lens, long max_q, long max_k, int causal, long window, float scale, Call& c) {
    if (type != SPANQR_BF16 && type != SPANQR_FP16) return error(SPANQR_EINVAL, "%s: the type must be bf16 or fp16", what);
    if (D < 8 || D > 128 || D % 8 != 0) return error(SPANQR_EINVAL, "%s: D = %ld (multiples of 8 up to 128)", what, D);
    if (B < 0 || Hk < 1 || G < 1 || Tq < 0 || Tk < 0 || B > INT_MAX / 2 || Hk > INT_MAX / G || (B + 1) > INT_MAX / Hk ||
        Tq >= MAX_ROWS / G || Tk >= MAX_ROWS || (Tq > 0 && Hk * G > INT_MAX / Tq))
        return error(SPANQR_EINVAL, "%s: B = %ld, heads = %ld x %ld, rows = %ld and %ld", what, B, Hk, G, Tq, Tk);
    if ((q_starts != nullptr) != (k_starts != nullptr)) return error(SPANQR_EINVAL, "%s: q_starts and k_starts belong together", what);
    if (k_lens != nullptr && q_starts != nullptr) return error(SPANQR_EINVAL, "%s: packed sequences have their lengths from k_starts", what);
    if (window < 0 || (window > 0 && !causal)) return error(SPANQR_EINVAL, "%s: a window needs causal, and one key at least", what);
    if (!(scale > 0.0f && scale * LOG2E < INFINITY)) return error(SPANQR_EINVAL, "%s: scale must be positive and finite", what);
    const bool packed = q_starts != nullptr;
    if (!packed || max_q < 1 || max_q > Tq) max_q = Tq;
    if (!packed || max_k < 1 || max_k > Tk) max_k = Tk;
    c.s = {(int)B, (int)Hk, (int)G, (int)D, Tq, Tk, q_starts, k_starts, k_lens, causal ? 1 : 0, (int)(window < MAX_ROWS ? window : MAX_ROWS),
           scale * LOG2E};
    c.rows = (packed ? 1 : B) * Tq * Hk * G;
    c.keys = (packed ? 1 : B) * Tk * Hk;
    const long q_all = Hk * count_of(packed, B, Tq * G, max_q * G, BLOCK), max_m = max_q * G;
    c.splits = B == 0 ? 1 : splits_of(q_all, max_k);
    c.few_keys = few_keys(Hk * count_of(packed, B, Tk, max_k, BLOCK), dkv_at_once(D));
    const long keys = c.few_keys ? BLOCK / 2 : BLOCK;
    c.q_splits = B == 0 || c.rows == 0 ? 1 : grad_splits_of(q_all, (max_k + TILE - 1) / TILE, dq_at_once(type, D), causal);
    c.kv_splits = B == 0 || c.keys == 0 ? 1 : grad_splits_of(Hk * count_of(packed, B, Tk, max_k, keys), (max_m + TILE - 1) / TILE, dkv_at_once(D), causal);
    c.tiles = tiles_of(packed, B, Hk, Tq * G, max_m, BLOCK, c.splits, c.splits == 1);
    c.q_tiles = tiles_of(packed, B, Hk, Tq * G, max_m, BLOCK, c.q_splits, c.q_splits == 1);
    c.k_tiles = tiles_of(packed, B, Hk, Tk, max_k, BLOCK, 1, false);
    c.kv_tiles = tiles_of(packed, B, Hk, Tk, max_k, keys, c.kv_splits, c.kv_splits == 1);
    if (c.tiles.n < 1 || c.q_tiles.n < 1 || c.k_tiles.n < 1 || c.kv_tiles.n < 1)
        return error(SPANQR_EINVAL, "%s: B = %ld sequences of %ld key heads are too many workgroups", what, B, Hk);
    return SPANQR_OK;
}

// two numbers a row, the maxima of fp16, and behind them (on 16 bytes) the parts
long maxima(const Call& c, const Tiles& t) { return (t.work == 0 ? (long)c.s.B * t.n : t.work) * c.s.Hk; }
long stat_bytes(const Call& c) { return 8 * c.rows + 4 * (maxima(c, c.q_tiles) + maxima(c, c.k_tiles)); }
long part_bytes(long rows, long splits, long D) { return splits == 1 ? 0 : 4 * rows * splits * D; }
long backward_bytes(const Call& c) {
    const long q = part_bytes(c.rows, c.q_splits, c.s.D), kv = 2 * part_bytes(c.keys, c.kv_splits, c.s.D);
    return q + kv == 0 ? stat_bytes(c) : (stat_bytes(c) + 15) / 16 * 16 + q + kv;
}

// strides: {batch, row, head}; keys: of k and v, whose tiles are of one head
int check_heads(const char* what, const char* name, const void* p, const long* strides, bool empty, bool keys, Heads& h) {
    if (empty) {
        h = {p, 0, 0, 0};
        return SPANQR_OK;
    }
    if (p == nullptr || strides == nullptr) return error(SPANQR_EINVAL, "%s: %s is missing", what, name);
    h = {p, strides[0], strides[1], strides[2]};
    if ((uintptr_t)p % 16 != 0 || h.batch % 8 != 0 || h.row % 8 != 0 || h.head % 8 != 0 || h.batch < 0 || h.row < 0 || h.head < 0 ||
        h.row >= MAX_STRIDE || (!keys && h.head >= MAX_STRIDE))
        return error(SPANQR_EINVAL, "%s: %s needs 16-byte alignment and strides that are multiples of 8, of rows%s below %ld", what, name,
                     keys ? "" : " and heads", MAX_STRIDE);
    return SPANQR_OK;
}
bool aligned(const void* p) { return (uintptr_t)p % 16 == 0; }

#define SPANQR_HEADS(LAUNCH)            \
    if (s.D <= 32) LAUNCH(32);          \
    else if (s.D <= 64) LAUNCH(64);     \
    else if (s.D <= 96) LAUNCH(96);     \
    else LAUNCH(128);

// extra: as in place_of
int grid_of(const Shape& s, const Tiles& t, bool extra, int splits) { return (t.work == 0 ? s.B + (extra ? 1 : 0) : 1) * s.Hk * t.n * splits; }

template <typename T>
void launch_forward(const ForwardArgs& a, hipStream_t st) {
    const Shape& s = a.s;
    const int grid = grid_of(s, a.tiles, s.q_starts != nullptr && a.splits == 1, a.splits);
#define LAUNCH(DP) k_forward<T, DP><<<grid, 64 * WAVES, 0, st>>>(a)
    SPANQR_HEADS(LAUNCH)
#undef LAUNCH
    if (a.splits > 1) {
        const int rows = (int)(a.rows < 65536 ? a.rows : 65536);
        if (a.splits <= 4 * WAVES)
            k_join<T, 4><<<rows, 64 * WAVES, 0, st>>>(a);
        else
            k_join<T, 16><<<rows, 64 * WAVES, 0, st>>>(a);
    }
}

template <typename T>
void launch_backward(const BackwardArgs& a, bool few_keys, hipStream_t st) {
    const Shape& s = a.s;
    const bool packed = s.q_starts != nullptr;
    if (std::is_same<T, fp16>::value && s.B > 0 && s.Tk > 0 && a.rows > 0)
        k_v_most<T><<<grid_of(s, a.k_tiles, false, 1), 64 * WAVES, 0, st>>>(a);
    if (a.rows > 0) {
#define LAUNCH(DP) k_dq<T, DP><<<grid_of(s, a.q_tiles, packed, a.q_splits), 64 * WAVES, 0, st>>>(a)
        SPANQR_HEADS(LAUNCH)
#undef LAUNCH
    }
    if (a.dk != nullptr && (packed || s.B > 0) && s.Tk > 0) {
        if (few_keys) {
#define LAUNCH(DP) k_dkv<T, DP, 2><<<grid_of(s, a.kv_tiles, packed, a.kv_splits), 64 * WAVES, 0, st>>>(a)
            SPANQR_HEADS(LAUNCH)
#undef LAUNCH
        } else {
#define LAUNCH(DP) k_dkv<T, DP, 1><<<grid_of(s, a.kv_tiles, packed, a.kv_splits), 64 * WAVES, 0, st>>>(a)
            SPANQR_HEADS(LAUNCH)
#undef LAUNCH
        }
    }
    if (a.q_splits > 1 || a.kv_splits > 1) {
        const long q_rows = packed ? s.Tq : s.B * s.Tq, k_rows = packed ? s.Tk : s.B * s.Tk, k_width = (long)s.Hk * s.D, q_width = k_width * s.G;
        PartsArgs p = {{{a.k_part, a.dk, s.k_starts, k_rows, k_width, a.kv_splits},
                        {a.v_part, a.dv, s.k_starts, k_rows, k_width, a.kv_splits},
                        {a.q_part, a.dq, s.q_starts, q_rows, q_width, a.q_splits}},
                       s.B};
        long most = 0;
        for (const Parts& x : p.of) most = x.splits > 1 && x.rows * x.width > most ? x.rows * x.width : most;
        const long grid = (most / 8 + 255) / 256;
        k_parts<T><<<dim3(grid < 2048 ? grid : 2048, 3), 256, 0, st>>>(p);
    }
}

}  // namespace

extern "C" {

long spanqr_attention_workspace(long B, long Hk, long G, long D, long Tq, long Tk, int packed, long max_q, long max_k) {
    Call c;
    const int none = 0;
    const int rc = check_shape("attention", SPANQR_BF16, B, Hk, G, D, Tq, Tk, packed ? &none : nullptr, packed ? &none : nullptr, nullptr,
                               max_q, max_k, 0, 0, 1.0f, c);
    if (rc != SPANQR_OK) return rc;
    return c.splits > 1 ? 4 * c.splits * c.rows * (D + 2) : 0;
}

int spanqr_attention(int type, long B, long Hk, long G, long D, long Tq, long Tk, const void* q, const long* q_strides, const void* k,
                     const long* k_strides, const void* v, const long* v_strides, const int* q_starts, const int* k_starts, const int* k_lens,
                     long max_q, long max_k, int causal, long window, float scale, void* out, float* lse, void* workspace, long workspace_bytes,
                     void* stream) {
    Call c;
    int rc = check_shape("attention", type, B, Hk, G, D, Tq, Tk, q_starts, k_starts, k_lens, max_q, max_k, causal, window, scale, c);
    if (rc != SPANQR_OK || c.rows == 0) return rc;
    ForwardArgs a = {};
    const bool none = Tk == 0 || (B == 0 && q_starts == nullptr);
    if ((rc = check_heads("attention", "q", q, q_strides, false, false, a.q)) != SPANQR_OK ||
        (rc = check_heads("attention", "k", k, k_strides, none, true, a.k)) != SPANQR_OK ||
        (rc = check_heads("attention", "v", v, v_strides, none, true, a.v)) != SPANQR_OK)
        return rc;
    if (out == nullptr || !aligned(out)) return error(SPANQR_EINVAL, "attention: out is missing or not on 16 bytes");
    const long need = c.splits > 1 ? 4 * c.splits * c.rows * (D + 2) : 0;
    if (need > 0 && (workspace == nullptr || !aligned(workspace) || workspace_bytes < need))
        return error(SPANQR_EINVAL, "attention: the workspace needs %ld bytes", need);
    a.s = c.s;
    a.out = out;
    a.lse = lse;
    a.tiles = c.tiles;
    a.splits = (int)c.splits;
    a.part = (float*)workspace;
    a.rows = c.rows;
    if (type == SPANQR_BF16)
        launch_forward<bf16>(a, (hipStream_t)stream);
    else
        launch_forward<fp16>(a, (hipStream_t)stream);
    return launched("attention");
}

long spanqr_attention_backward_workspace(long B, long Hk, long G, long D, long Tq, long Tk, int packed, long max_q, long max_k) {
    Call c;
    const int none = 0;
    const int rc = check_shape("attention_backward", SPANQR_BF16, B, Hk, G, D, Tq, Tk, packed ? &none : nullptr, packed ? &none : nullptr,
                               nullptr, max_q, max_k, 1, 0, 1.0f, c);   // (causal ones in bf16 have the most parts)
    return rc != SPANQR_OK ? rc : backward_bytes(c);
}

int spanqr_attention_backward(int type, long B, long Hk, long G, long D, long Tq, long Tk, const void* dout, const long* dout_strides,
                              const void* q, const long* q_strides, const void* k, const long* k_strides, const void* v,
                              const long* v_strides, const void* out, const long* out_strides, const float* lse, const int* q_starts,
                              const int* k_starts, const int* k_lens, long max_q, long max_k, int causal, long window, float scale, void* dq, void* dk,
                              void* dv, void* workspace, long workspace_bytes, void* stream) {
    const char* what = "attention_backward";
    Call c;
    int rc = check_shape(what, type, B, Hk, G, D, Tq, Tk, q_starts, k_starts, k_lens, max_q, max_k, causal, window, scale, c);
    if (rc != SPANQR_OK) return rc;
    const bool packed = q_starts != nullptr, no_q = c.rows == 0, no_k = Tk == 0 || (B == 0 && !packed);
    BackwardArgs a = {};
    if ((rc = check_heads(what, "q", q, q_strides, no_q, false, a.q)) != SPANQR_OK ||
        (rc = check_heads(what, "k", k, k_strides, no_k, true, a.k)) != SPANQR_OK ||
        (rc = check_heads(what, "v", v, v_strides, no_k, true, a.v)) != SPANQR_OK ||
        (rc = check_heads(what, "out", out, out_strides, no_q, false, a.out)) != SPANQR_OK ||
        (rc = check_heads(what, "dout", dout, dout_strides, no_q, false, a.dout)) != SPANQR_OK)
        return rc;
    if ((dk != nullptr) != (dv != nullptr) || !aligned(dq) || !aligned(dk) || !aligned(dv))
        return error(SPANQR_EINVAL, "%s: dk and dv belong together, and gradients lie on 16 bytes", what);
    if (c.rows > 0 && lse == nullptr) return error(SPANQR_EINVAL, "%s: lse is missing", what);
    const long need = backward_bytes(c);
    if (need > 0 && (workspace == nullptr || !aligned(workspace) || workspace_bytes < need))
        return error(SPANQR_EINVAL, "%s: the workspace needs %ld bytes", what, need);
    if (no_q && (no_k || dk == nullptr)) return SPANQR_OK;
    a.s = c.s;
    a.lse = lse;
    a.dq = dq;
    a.dk = dk;
    a.dv = dv;
    a.stat = (float*)workspace;
    a.rows = c.rows;
    a.q_tiles = c.q_tiles;
    a.k_tiles = c.k_tiles;
    a.kv_tiles = c.kv_tiles;
    a.scale = scale;
    a.v_most = a.stat + 2 * c.rows;
    a.d_most = a.v_most + maxima(c, c.k_tiles);
    a.q_splits = dq != nullptr ? (int)c.q_splits : 1;
    a.kv_splits = dk != nullptr ? (int)c.kv_splits : 1;
    a.q_part = (float*)((char*)workspace + (stat_bytes(c) + 15) / 16 * 16);
    a.k_part = a.q_part + part_bytes(c.rows, c.q_splits, D) / 4;
    a.v_part = a.k_part + part_bytes(c.keys, c.kv_splits, D) / 4;
    if (type == SPANQR_BF16)
        launch_backward<bf16>(a, c.few_keys, (hipStream_t)stream);
    else
        launch_backward<fp16>(a, c.few_keys, (hipStream_t)stream);
    return launched(what);
}

}  // extern "C"
