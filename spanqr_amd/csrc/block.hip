// block.hip -- what stands between two blocks of a model: the norm behind a block, its gate, dropout, the scaled addition to
// the stream and the norm in front of the next block, in one pass, with its gradient; and dropout alone.
//
//   n1 = x s1, s1 = (sum_j x_j^2 / D + eps)^(-1/2);  t = n1 w1 act(g);  h = round(r + a k t), k = 0 or 1 / (1 - p)
//   n2 = h s2, s2 = (sum_j h_j^2 / D + eps)^(-1/2);  y = n2 w2
//   gradient: dr = s2 (dy w2 - n2 mean(dy w2 n2)) + dh,  v = k dr,  q = v w1 act(g)
//             dx = a s1 (q - n1 mean(q n1)),  dg = a v n1 w1 act'(g)
//             dw1 = a sum over rows of v act(g) n1,  dw2 = sum over rows of dy n2,  da = sum of q n1
//   act(g) = g, 1 / (1 + exp(-g)), or g / (1 + exp(-g)); 1 without a gate
//
// Bound by memory: rows of up to 8192 elements are read once and each output written once, the row stays in registers between the
// two sums (threads and pieces as in norm.hip). Between them would be h, t, n1, dt and the mask in memory if these were operators of
// their own. Longer rows are read two or three times, from the caches behind the first one (k_block_long, k_block_grad_long).
// Sums are fp32 in a fixed order. Within a row: per thread over at most 16 elements, or the D / 8192 pieces of eight (up to 2048) of a
// long one, then a tree. Over rows, for the weights and the scale: a thread's rows one after the other (rows / 256 at
// most), up to 16 groups, then at most 24 of up to 1536 parts in each of 64 sums, and a tree: rows / 256 + 50 steps of 2^-24 of what is
// added up, at most. 16384 x 2048 bf16 with gate and
// dropout: forward 61 us for 0.34 GB, gradient 91 for 0.54 GB and k_block_sums 7, with the 256 MB cache's help above a large
// copy's 5.2 TB/s; without dropout's ten rounds of multiplications 161 us in all instead of 169.
#include "host.h"
#include "random.h"
#include "rows.h"

using namespace spanqr_dev;
using spanqr_host::error;
using spanqr_host::launched;

namespace {

struct BlockArgs {
    long rows, D, ldx, ldr, ldg;
    const void *x, *residual, *gate, *w1, *w2;   // gate and the weights may be null
    int wtype, act;
    float eps, scale;
    const float* scale_at;                       // read instead of scale where it is not null
    Dropout drop;
    void *h, *y;
    bool past;                                   // the outputs do not fit the caches
};

struct BlockGradArgs {
    long rows, D, lddy, lddh, ldx, ldh, ldg;
    const void *dy, *dh, *x, *h, *gate, *w1, *w2;   // dy or dh, gate and the weights may be null
    int wtype, act;
    float eps, scale;
    const float* scale_at;
    Dropout drop;
    void *dx, *dr, *dg;                          // dg null without a gate
    bool past;
    float* part;                                 // [gridDim.x][2 D + 1] sums over the workgroup's rows for dw1, dw2, da, or null
};

// the factor of what is added to the stream, in a scalar register
template <typename ARGS>
__device__ __forceinline__ float factor_of(const ARGS& p) {
    const float a = p.scale_at != nullptr ? *p.scale_at : p.scale;
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, a)));
}

// Both weights of a thread's columns in fp32 in LDS, each thread's own words: read from memory in every row they would be two
// more latencies, in registers 16 a piece. 64 bytes for each thread and piece.
template <int NCH>
struct Weights {
    float4* at;
    __device__ __forceinline__ Weights(float4* lds, const void* w1, const void* w2, int type, long D, int lane, int size) : at(lds + threadIdx.x) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const long from = 8l * (lane + c * size);
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                float w[8];
                load_weight(which ? w2 : w1, type, from, inside(D, from), w);
                at[(4 * c + 2 * which) * blockDim.x] = make_float4(w[0], w[1], w[2], w[3]);
                at[(4 * c + 2 * which + 1) * blockDim.x] = make_float4(w[4], w[5], w[6], w[7]);
            }
        }
    }
    __device__ __forceinline__ void get(int which, int c, float (&w)[8]) const {
        const float4 a = at[(4 * c + 2 * which) * blockDim.x], b = at[(4 * c + 2 * which + 1) * blockDim.x];
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
    }
};

// 1 / (1 + exp(-g)): in fp32's full precision, or for what is rounded to 16 bits from 2^t, t = -g log2 e. The product's rounding
// makes that 2^-20 of itself for |g| up to 16, of which bf16 (2^-9 at best) sees nothing; fp16 has it taken out.
// e: exp(-g)
template <typename T>
__device__ __forceinline__ float sigmoid(float g, float& e) {
    if constexpr (sizeof(T) == 4) {
        e = expf(-g);
        return 1.0f / (1.0f + e);
    }
    constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
    const float t = -LOG2E * g;
    e = __builtin_amdgcn_exp2f(t);
    if constexpr (std::is_same<T, fp16>::value) {
        const float left = fmaf(-LOG2E, g, -t);
        e = fabsf(g) < 88.0f ? fmaf(e, LN2 * left, e) : e;   // (beyond: infinite, or as good as 0)
    }
    return __builtin_amdgcn_rcpf(1.0f + e);
}
template <typename T>
__device__ __forceinline__ float sigmoid(float g) {
    float e;
    return sigmoid<T>(g, e);
}
// s = sigmoid(g), and 1 - s as exp(-g) s, which keeps what the difference loses where s is next to 1 (half a percent of it at g = 12);
// 0 where exp(-g) overflows, and s with it is 0. (With a choice by g's sign, for the sigmoid's slope alone, the compiler took 171
// registers instead of 160: 131 -> 159 us at 16384 x 2048 bf16 without a gate, both ways.)
template <typename T>
__device__ __forceinline__ void sigmoid_and_rest(float g, float& s, float& rest) {
    float e;
    s = sigmoid<T>(g, e);
    rest = fminf(e, 0x1.fffffep127f) * s;
}

// v act(g)
template <typename T>
__device__ __forceinline__ void times_gate(int act, const float (&g)[8], float (&v)[8]) {
    if (act == SPANQR_GATE_LINEAR) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= g[i];
    } else if (act == SPANQR_GATE_SIGMOID) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= sigmoid<T>(g[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= g[i] * sigmoid<T>(g[i]);
    }
}
// v act(g) in v, and u act'(g) in g
template <typename T>
__device__ __forceinline__ void gate_slope(int act, float (&g)[8], float (&v)[8], const float (&u)[8]) {
    if (act == SPANQR_GATE_LINEAR) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] *= g[i];
            g[i] = u[i];
        }
    } else if (act == SPANQR_GATE_SIGMOID) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float s, rest;
            sigmoid_and_rest<T>(g[i], s, rest);
            v[i] *= s;
            g[i] = u[i] * (s * rest);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float s, rest;
            sigmoid_and_rest<T>(g[i], s, rest);
            const float a = g[i] * s;
            v[i] *= a;
            g[i] = u[i] * (s + a * rest);
        }
    }
}

template <typename T, int GROUP, int NCH, int WHOLE>
__global__ __launch_bounds__(Group<GROUP>::MOST) void k_block(const BlockArgs p) {
    typedef Group<GROUP> G;
    __shared__ float slot[2][2][1][16];   // both sums', by turns
    extern __shared__ float4 weights[];
    const int lane = G::lane(), size = G::size();
    const Weights<NCH> weight(weights, p.w1, p.w2, p.wtype, p.D, lane, size);
    const float scale = factor_of(p);
    const uint64_t key = p.drop.key();
    // (a load under a condition would be waited for before the next one: without a gate x is read again, from the cache)
    const void* gate = p.gate != nullptr ? p.gate : p.x;
    const long ldg = p.gate != nullptr ? p.ldg : p.ldx;
    int turn = 0;
    for (long base = (long)blockIdx.x * G::rows(); base < p.rows; base += (long)gridDim.x * G::rows(), turn ^= 1) {
        const long row = base + G::index();
        const bool on = row < p.rows;   // the group's lanes all take part in the reductions
        const long from = on ? row : base;
        Pack8<T> kx[NCH], kr[NCH], kg[NCH];
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const long at = 8l * (lane + c * size);
            const int n = inside(p.D, at);
            kx[c] = piece<WHOLE>((const T*)p.x + from * p.ldx, p.D, at, n);
            kr[c] = piece<WHOLE>((const T*)p.residual + from * p.ldr, p.D, at, n);
            kg[c] = piece<WHOLE>((const T*)gate + from * ldg, p.D, at, n);
        }
        float sum[1] = {0.0f};
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            float x[8];
            settle<WHOLE>(kx[c], on ? inside(p.D, 8l * (lane + c * size)) : 0, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[0] = fmaf(x[i], x[i], sum[0]);
        }
        G::sum(sum, slot[turn][0]);
        const float s1 = rsqrtf(sum[0] / (float)p.D + p.eps);
        float h[NCH][8];
        sum[0] = 0.0f;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const long at = 8l * (lane + c * size);
            const int n = on ? inside(p.D, at) : 0;
            float x[8], w[8];
            settle<WHOLE>(kx[c], n, x);
            settle<WHOLE>(kr[c], n, h[c]);
            weight.get(0, c, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * s1 * w[i];
            if (p.gate != nullptr) {
                float g[8];
                settle<WHOLE>(kg[c], n, g);
                times_gate<T>(p.act, g, x);
            }
            p.drop.thin(key, row, lane + c * size, x);
            // the stream is rounded as it is kept; the norm is of the rounded values
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                h[c][i] = i < n ? (float)(T)fmaf(scale, x[i], h[c][i]) : 0.0f;
                sum[0] = fmaf(h[c][i], h[c][i], sum[0]);
            }
            store8((T*)p.h + row * p.D + at, n, h[c], p.past);
        }
        G::sum(sum, slot[turn][1]);
        const float s2 = rsqrtf(sum[0] / (float)p.D + p.eps);
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const long at = 8l * (lane + c * size);
            const int n = on ? inside(p.D, at) : 0;
            float w[8];
            weight.get(1, c, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[c][i] = h[c][i] * s2 * w[i];
            store8((T*)p.y + row * p.D + at, n, h[c], p.past);
        }
    }
}

// Rows longer than 8192: one workgroup a row, x and h read twice (from the cache the second time). Keeping h of up to 24576
// elements in registers took 235 us where this takes 207 (4096 x 14336 bf16).
template <typename T>
__global__ __launch_bounds__(1024) void k_block_long(const BlockArgs p) {
    __shared__ float slot[3][1][16];
    typedef Group<0> G;
    const float scale = factor_of(p);
    const uint64_t key = p.drop.key();
    int turn = 0;
    for (long row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const T* x = (const T*)p.x + row * p.ldx;
        T* h = (T*)p.h + row * p.D;
        float sum[1] = {0.0f}, v[8], w[8], u[8];
#pragma unroll 2
        for (long at = 8l * threadIdx.x; at < p.D; at += 8192) {
            settle8(fetch8(x, p.D, at), inside(p.D, at), v);
            float part = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) part = fmaf(v[i], v[i], part);
            sum[0] += part;
        }
        G::sum(sum, slot[turn]);
        const float s1 = rsqrtf(sum[0] / (float)p.D + p.eps);
        sum[0] = 0.0f;
        for (long at = 8l * threadIdx.x; at < p.D; at += 8192) {
            const int n = inside(p.D, at);
            const Pack8<T> kx = fetch8(x, p.D, at), kr = fetch8((const T*)p.residual + row * p.ldr, p.D, at);
            settle8(kx, n, v);
            load_weight(p.w1, p.wtype, at, n, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = v[i] * s1 * w[i];
            if (p.gate != nullptr) {
                settle8(fetch8((const T*)p.gate + row * p.ldg, p.D, at), n, w);
                times_gate<T>(p.act, w, v);
            }
            p.drop.thin(key, row, at >> 3, v);
            settle8(kr, n, u);
            float part = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                u[i] = i < n ? (float)(T)fmaf(scale, v[i], u[i]) : 0.0f;
                part = fmaf(u[i], u[i], part);
            }
            store8(h + at, n, u);
            sum[0] += part;
        }
        G::sum(sum, slot[2]);   // (the next row's first barrier stands between its reads and the next writes)
        const float s2 = rsqrtf(sum[0] / (float)p.D + p.eps);
        // a thread reads back only what it wrote itself
        for (long at = 8l * threadIdx.x; at < p.D; at += 8192) {
            const int n = inside(p.D, at);
            load8(h + at, n, v);
            load_weight(p.w2, p.wtype, at, n, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = v[i] * s2 * w[i];
            store8((T*)p.y + row * p.D + at, n, v, p.past);
        }
    }
}

// The weights' gradients are sums over rows: a workgroup keeps its rows' part in registers (each thread always holds the same
// columns), adds its groups through LDS and writes one row of partial sums; k_block_sums adds those.
template <typename T, int GROUP, int NCH, int WHOLE>
__global__ __launch_bounds__(GROUP ? 256 : 512) void k_block_grad(const BlockGradArgs p) {
    typedef Group<GROUP> G;
    __shared__ float slot[2][3][16], slot2[2][1][16];
    constexpr int ROWS = GROUP ? 256 / GROUP : 1;
    __shared__ float add[ROWS > 1 ? (ROWS - 1) * GROUP * NCH * 16 : 1];
    __shared__ float add_scale[ROWS];
    extern __shared__ float4 weights[];
    const int lane = G::lane(), group = G::index(), size = G::size();
    const Weights<NCH> weight(weights, p.w1, p.w2, p.wtype, p.D, lane, size);
    const float scale = factor_of(p);
    const uint64_t key = p.drop.key();
    float dw1[NCH][8], dw2[NCH][8], da = 0.0f;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) dw1[c][i] = dw2[c][i] = 0.0f;
    // (a load under a condition would be waited for before the next one: for what is absent h is read again, from the cache)
    const void *dy = p.dy != nullptr ? p.dy : p.h, *dh = p.dh != nullptr ? p.dh : p.h, *gate = p.gate != nullptr ? p.gate : p.h;
    const long lddy = p.dy != nullptr ? p.lddy : p.ldh, lddh = p.dh != nullptr ? p.lddh : p.ldh, ldg = p.gate != nullptr ? p.ldg : p.ldh;
    struct Row {
        Pack8<T> x[NCH], h[NCH], y[NCH], d[NCH], g[NCH];
    };
    auto fetch = [&](long base, Row& k) {
        const long from = base + group < p.rows ? base + group : base;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const long at = 8l * (lane + c * size);
            const int n = inside(p.D, at);
            k.x[c] = piece<WHOLE>((const T*)p.x + from * p.ldx, p.D, at, n);
            k.h[c] = piece<WHOLE>((const T*)p.h + from * p.ldh, p.D, at, n);
            k.y[c] = piece<WHOLE>((const T*)dy + from * lddy, p.D, at, n);
            k.d[c] = piece<WHOLE>((const T*)dh + from * lddh, p.D, at, n);
            k.g[c] = piece<WHOLE>((const T*)gate + from * ldg, p.D, at, n);
        }
    };
    const long step = (long)gridDim.x * ROWS;
    int turn = 0;
    Row k, next;
    if ((long)blockIdx.x * ROWS < p.rows) fetch((long)blockIdx.x * ROWS, next);
    for (long base = (long)blockIdx.x * ROWS; base < p.rows; base += step, turn ^= 1) {
        const long row = base + group;
        const bool on = row < p.rows;
        k = next;
        if (base + step < p.rows) fetch(base + step, next);
        float sum[3] = {0.0f, 0.0f, 0.0f};   // of x^2, h^2 and dy w2 h
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const long at = 8l * (lane + c * size);
            const int n = on ? inside(p.D, at) : 0;
            float x[8], h[8], u[8], w[8];
            settle<WHOLE>(k.x[c], n, x);
            settle<WHOLE>(k.h[c], p.dy != nullptr ? n : 0, h);
            settle<WHOLE>(k.y[c], p.dy != nullptr ? n : 0, u);
            weight.get(1, c, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sum[0] = fmaf(x[i], x[i], sum[0]);
                sum[1] = fmaf(h[i], h[i], sum[1]);
                sum[2] = fmaf(u[i] * w[i], h[i], sum[2]);
            }
        }
        G::sum(sum, slot[turn]);
        // a group without a row adds zeros, also where eps is 0
        const float s1 = on ? rsqrtf(sum[0] / (float)p.D + p.eps) : 0.0f;
        const float s2 = on && p.dy != nullptr ? rsqrtf(sum[1] / (float)p.D + p.eps) : 0.0f;   // (without dy: dh alone)
        const float m2 = s2 * sum[2] / (float)p.D;   // the mean of dy w2 n2
        float q[NCH][8], last[1] = {0.0f};
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            again(k.x[c]);   // (packed they take half the registers until here)
            again(k.h[c]);
            again(k.y[c]);
            const long at = 8l * (lane + c * size);
            const int n = on ? inside(p.D, at) : 0;
            float a[8], b[8], w[8], d[8];
            settle<WHOLE>(k.h[c], p.dy != nullptr ? n : 0, a);   // (without dy h counts nothing, whatever it holds)
            settle<WHOLE>(k.y[c], p.dy != nullptr ? n : 0, b);
            settle<WHOLE>(k.d[c], p.dh != nullptr ? n : 0, d);
            weight.get(1, c, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float n2 = a[i] * s2;
                dw2[c][i] = fmaf(b[i], n2, dw2[c][i]);
                d[i] = fmaf(s2, b[i] * w[i] - n2 * m2, d[i]);
            }
            store8((T*)p.dr + row * p.D + at, n, d, p.past);
            p.drop.thin(key, row, lane + c * size, d);
            settle<WHOLE>(k.x[c], n, a);
            weight.get(0, c, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                d[i] = i < n ? d[i] : 0.0f;
                a[i] *= s1;
            }
            if (p.gate != nullptr) {
                float g[8];
                settle<WHOLE>(k.g[c], n, g);
#pragma unroll
                for (int i = 0; i < 8; ++i) b[i] = scale * d[i] * a[i] * w[i];
                gate_slope<T>(p.act, g, d, b);
                store8((T*)p.dg + row * p.D + at, n, g, p.past);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                dw1[c][i] = fmaf(d[i], a[i], dw1[c][i]);
                q[c][i] = i < n ? d[i] * w[i] : 0.0f;
                last[0] = fmaf(q[c][i], a[i], last[0]);
            }
        }
        G::sum(last, slot2[turn]);
        const float m1 = last[0] / (float)p.D;   // the mean of q n1
        if (lane == 0) da += last[0];
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            again(k.x[c]);
            const long at = 8l * (lane + c * size);
            const int n = on ? inside(p.D, at) : 0;
            float x[8];
            settle<WHOLE>(k.x[c], n, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = scale * s1 * (q[c][i] - x[i] * s1 * m1);
            store8((T*)p.dx + row * p.D + at, n, x, p.past);
        }
    }
    if (p.part == nullptr) return;
    if constexpr (ROWS > 1) {
        if (group > 0) {
#pragma unroll
            for (int c = 0; c < NCH; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    add[((group - 1) * NCH * 16 + c * 16 + i) * GROUP + lane] = dw1[c][i];
                    add[((group - 1) * NCH * 16 + c * 16 + 8 + i) * GROUP + lane] = dw2[c][i];
                }
        }
        if (lane == 0) add_scale[group] = da;
        __syncthreads();
        if (group > 0) return;
        for (int g = 0; g < ROWS - 1; ++g) {
#pragma unroll
            for (int c = 0; c < NCH; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    dw1[c][i] += add[(g * NCH * 16 + c * 16 + i) * GROUP + lane];
                    dw2[c][i] += add[(g * NCH * 16 + c * 16 + 8 + i) * GROUP + lane];
                }
            da += add_scale[g + 1];
        }
    }
    float* part = p.part + blockIdx.x * (2 * p.D + 1);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const long at = 8l * (lane + c * size);
#pragma unroll
        for (int i = 0; i < 8; ++i) dw1[c][i] *= scale;
        store8(part + at, inside(p.D, at), dw1[c]);
        store8(part + p.D + at, inside(p.D, at), dw2[c]);
    }
    if (lane == 0) part[2 * p.D] = da;
}

// The gradient of rows longer than 8192: one workgroup a row, which is read for each of three steps (from L2 behind the first
// one). The sums for the weights are in LDS (up to LONG_LDS columns), or in the partial sums' own memory; a thread's own words
// either way. With the sums in registers and q kept in LDS for the third step it took 1082 us (4096 x 14336 bf16: they spill).
constexpr int LONG_LDS = 18432;
template <typename T, bool IN_LDS>
__global__ __launch_bounds__(1024) void k_block_grad_long(const BlockGradArgs p) {
    __shared__ float slot[2][3][16], slot2[2][1][16];
    __shared__ __attribute__((aligned(16))) float add[IN_LDS ? 2 * LONG_LDS : 4];
    typedef Group<0> G;
    const float scale = factor_of(p);
    const uint64_t key = p.drop.key();
    float* part = p.part == nullptr ? nullptr : p.part + blockIdx.x * (2 * p.D + 1);
    const void *dy = p.dy != nullptr ? p.dy : p.h, *dh = p.dh != nullptr ? p.dh : p.h, *gate = p.gate != nullptr ? p.gate : p.h;
    const long lddy = p.dy != nullptr ? p.lddy : p.ldh, lddh = p.dh != nullptr ? p.lddh : p.ldh, ldg = p.gate != nullptr ? p.ldg : p.ldh;
    const int n_y = p.dy != nullptr ? 8 : 0, n_d = p.dh != nullptr ? 8 : 0, t = threadIdx.x;
    // adds v to the sums of piece `at`: the weight behind the block (0) or in front of the next one (1)
    auto sums = [&](int which, long at, int n, bool start, const float (&v)[8]) {
        float* mine = IN_LDS ? add + which * LONG_LDS + at : part + which * p.D + at;
        if (!IN_LDS && part == nullptr) return;
        float old[8];
        load8(mine, start ? 0 : n, old);
#pragma unroll
        for (int i = 0; i < 8; ++i) old[i] += v[i];
        store8(mine, n, old);
    };
    float da = 0.0f;
    int turn = 0;
    for (long row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const T* xr = (const T*)p.x + row * p.ldx;
        const T* hr = (const T*)p.h + row * p.ldh;
        const T* yr = (const T*)dy + row * lddy;
        const T* dr = (const T*)dh + row * lddh;
        const T* gr = (const T*)gate + row * ldg;
        float sum[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll 2
        for (long at = 8l * t; at < p.D; at += 8192) {
            const int n = inside(p.D, at);
            const Pack8<T> kx = fetch8(xr, p.D, at), kh = fetch8(hr, p.D, at), ky = fetch8(yr, p.D, at);
            float a[8], b[8], w[8], e = 0.0f, f = 0.0f, g = 0.0f;
            settle8(kx, n, a);
#pragma unroll
            for (int i = 0; i < 8; ++i) e = fmaf(a[i], a[i], e);
            settle8(kh, n < n_y ? n : n_y, a);
            settle8(ky, n < n_y ? n : n_y, b);
            load_weight(p.w2, p.wtype, at, n, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                f = fmaf(a[i], a[i], f);
                g = fmaf(b[i] * w[i], a[i], g);
            }
            sum[0] += e;
            sum[1] += f;
            sum[2] += g;
        }
        G::sum(sum, slot[turn]);
        const float s1 = rsqrtf(sum[0] / (float)p.D + p.eps);
        const float s2 = p.dy != nullptr ? rsqrtf(sum[1] / (float)p.D + p.eps) : 0.0f;   // (without dy: dh alone)
        const float m2 = s2 * sum[2] / (float)p.D;
        // q and n1 of a piece; in the first of two steps with everything else that the piece gives
        auto piece_of = [&](long at, bool first, float (&q)[8], float (&n1)[8]) __attribute__((always_inline)) {
            const int n = inside(p.D, at);
            const Pack8<T> kh = fetch8(hr, p.D, at), ky = fetch8(yr, p.D, at), kd = fetch8(dr, p.D, at), kx = fetch8(xr, p.D, at),
                           kg = fetch8(gr, p.D, at);
            float a[8], b[8], w[8];
            settle8(kh, n < n_y ? n : n_y, a);
            settle8(ky, n < n_y ? n : n_y, b);
            settle8(kd, n < n_d ? n : n_d, q);
            load_weight(p.w2, p.wtype, at, n, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                a[i] *= s2;
                q[i] = fmaf(s2, b[i] * w[i] - a[i] * m2, q[i]);
                a[i] *= b[i];
            }
            if (first) {
                store8((T*)p.dr + row * p.D + at, n, q, p.past);
                sums(1, at, n, row == blockIdx.x, a);
            }
            p.drop.thin(key, row, at >> 3, q);
            settle8(kx, n, n1);
            load_weight(p.w1, p.wtype, at, n, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                q[i] = i < n ? q[i] : 0.0f;
                n1[i] *= s1;
            }
            if (p.gate != nullptr) {
                settle8(kg, n, b);
#pragma unroll
                for (int i = 0; i < 8; ++i) a[i] = scale * q[i] * n1[i] * w[i];
                gate_slope<T>(p.act, b, q, a);
                if (first) store8((T*)p.dg + row * p.D + at, n, b, p.past);
            }
            if (first) {
#pragma unroll
                for (int i = 0; i < 8; ++i) a[i] = scale * q[i] * n1[i];
                sums(0, at, n, row == blockIdx.x, a);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = i < n ? q[i] * w[i] : 0.0f;
        };
        float last[1] = {0.0f}, q[8], n1[8];
        for (long at = 8l * t; at < p.D; at += 8192) {
            piece_of(at, true, q, n1);
            float a = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) a = fmaf(q[i], n1[i], a);
            last[0] += a;
        }
        G::sum(last, slot2[turn]);
        const float m1 = last[0] / (float)p.D;
        da += last[0];
        for (long at = 8l * t; at < p.D; at += 8192) {
            piece_of(at, false, q, n1);
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = scale * s1 * (q[i] - n1[i] * m1);
            store8((T*)p.dx + row * p.D + at, inside(p.D, at), q, p.past);
        }
    }
    if (part == nullptr) return;
    if constexpr (IN_LDS) {
        for (long at = 8l * t; at < p.D; at += 8192)
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                float v[8];
                load8(add + which * LONG_LDS + at, inside(p.D, at), v);
                store8(part + which * p.D + at, inside(p.D, at), v);
            }
    }
    if (t == 0) part[2 * p.D] = da;
}

// columns [0, D) of the parts are dw1's, [D, 2 D) dw2's, the last is da's: 16 columns a workgroup, 64 threads a column, added in
// a fixed order
__global__ __launch_bounds__(1024) void k_block_sums(const float* part, int parts, long D, void* dw1, void* dw2, int wtype, float* da) {
    __shared__ float add[64][17];
    const long all = 2 * D + 1;
    const int col = threadIdx.x & 15, at = threadIdx.x >> 4;
    long d = 16l * blockIdx.x + col;
    float sum = 0.0f;
    if (d < all) {
#pragma unroll 8
        for (int i = at; i < parts; i += 64) sum += part[i * all + d];
    }
    add[at][col] = sum;
    __syncthreads();
    // a wavefront a column
    d = 16l * blockIdx.x + (threadIdx.x >> 6);
    sum = reduce_lanes<64, Sum>(add[threadIdx.x & 63][threadIdx.x >> 6]);
    if ((threadIdx.x & 63) != 0 || d >= all) return;
    if (d == 2 * D) {
        if (da != nullptr) *da = sum;
        return;
    }
    void* dw = d < D ? dw1 : dw2;
    if (dw == nullptr) return;
    if (d >= D) d -= D;
    if (wtype == SPANQR_BF16)
        ((bf16*)dw)[d] = (bf16)sum;
    else if (wtype == SPANQR_FP16)
        ((fp16*)dw)[d] = (fp16)sum;
    else
        ((float*)dw)[d] = sum;
}

// outputs of more than the eight L2s' 32 MB are written past them
bool past_caches(long rows, long D, long bytes) { return rows * D * bytes > 32l << 20; }

// Dropout alone: a workgroup takes DROP_PIECES neighbouring pieces at a time, a thread every 256th of them, so that its loads
// are under way together. pieces: of a row. 16384 x 5120 bf16: 70 us, 4.8 TB/s.
constexpr int DROP_PIECES = 512;
template <typename T>
__global__ __launch_bounds__(256) void k_dropout(long rows, long D, uint32_t pieces, const T* x, long ldx, Dropout drop, T* y, bool past) {
    constexpr int N = DROP_PIECES / 256;
    const uint64_t key = drop.key();
    const long all = rows * pieces;
    for (long first = (long)blockIdx.x * DROP_PIECES; first < all; first += (long)gridDim.x * DROP_PIECES) {
        const long row0 = first / pieces;
        const uint32_t col0 = (uint32_t)(first - row0 * pieces);
        Pack8<T> k[N];
        long row[N], at[N];
        int n[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t t = threadIdx.x + 256 * i, to = col0 + t, over = to / pieces;
            const bool on = first + t < all;
            row[i] = on ? row0 + over : row0;
            at[i] = 8l * (on ? to - over * pieces : col0);
            n[i] = on ? inside(D, at[i]) : 0;
            k[i] = D >= 8 ? fetch8(x + row[i] * ldx, D, at[i]) : piece<false>(x + row[i] * ldx, D, at[i], n[i]);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float v[8];
            if (D >= 8)
                settle8(k[i], n[i], v);
            else
                settle<false>(k[i], n[i], v);
            drop.thin(key, row[i], at[i] >> 3, v);
            store8(y + row[i] * D + at[i], n[i], v, past);
        }
    }
}

constexpr long LONG_ROW = 8192;   // longest row that stays in registers
constexpr long MAX_D = 1l << 24;
constexpr long MAX_DROP_D = 1l << 32;   // dropout alone

Split split_of(long rows, long D) {
    const long pieces = (D + 7) / 8;
    if (D <= 128) return {16, 1, false};
    if (D <= 512) return {64, 1, false};
    const int nch = D <= 2048 || (rows <= 512 && D <= 8192) ? 1 : 2;
    return {(int)(((pieces + nch - 1) / nch + 63) / 64 * 64), nch, true};
}
Split grad_split_of(long D) {
    const long pieces = (D + 7) / 8;
    if (D <= 128) return {16, 1, false};
    if (D <= 512) return {64, 1, false};
    const int nch = D <= 4096 ? 1 : 2;
    return {(int)(((pieces + nch - 1) / nch + 63) / 64 * 64), nch, true};
}

// The gradient's workgroups, and so rows of partial sums: as many as the compute units hold at once (12 wavefronts of one
// piece a thread each, 8 of two), but where there are few rows at least four for each, since each workgroup ends with a row of sums
// that is written and read again. Forward and gradient in us with 768 / 1536: 16384 x 1024 bf16 115 / 103, 3001 x 769 fp32 37 / 43.
int grad_parts(long rows, long D) {
    if (D > LONG_ROW) return (int)(rows < 256 ? rows : 256);
    const Split s = grad_split_of(D);
    const long most = !s.block ? 1024 : s.group <= 128 ? 1536 : s.group <= 256 ? 768 : 256, few = rows / 4 > 256 ? rows / 4 : 256;
    return grid_of(rows, s, (int)(most < few ? most : few));
}

#define SPANQR_BLOCK_SPLITS(LAUNCH)                       \
    if (s.block && s.nch == 2) {                          \
        if (p.D % 8 == 0) LAUNCH(0, 2, 2);                \
        else LAUNCH(0, 2, 1);                             \
    } else if (s.block) {                                 \
        if (p.D % 8 == 0) LAUNCH(0, 1, 2);                \
        else LAUNCH(0, 1, 1);                             \
    } else if (s.group == 64) {                           \
        if (p.D % 8 == 0) LAUNCH(64, 1, 2);               \
        else LAUNCH(64, 1, 1);                            \
    } else if (p.D >= 8) {                                \
        if (p.D % 8 == 0) LAUNCH(16, 1, 2);               \
        else LAUNCH(16, 1, 1);                            \
    } else {                                              \
        LAUNCH(16, 1, 0);                                 \
    }

template <typename T>
void launch_block(const BlockArgs& p, hipStream_t st) {
    if (p.D > LONG_ROW) {
        k_block_long<T><<<(int)(p.rows < 1024 ? p.rows : 1024), 1024, 0, st>>>(p);
        return;
    }
    const Split s = split_of(p.rows, p.D);
    const int grid = grid_of(p.rows, s, s.block ? 1024 : 2048);
    const int threads = s.block ? s.group : 256;
#define LAUNCH(G, C, W) k_block<T, G, C, W><<<grid, threads, 64 * C * threads, st>>>(p)
    SPANQR_BLOCK_SPLITS(LAUNCH)
#undef LAUNCH
}

template <typename T>
void launch_grad(const BlockGradArgs& p, int grid, hipStream_t st) {
    if (p.D > LONG_ROW) {
        if (p.D <= LONG_LDS)
            k_block_grad_long<T, true><<<grid, 1024, 0, st>>>(p);
        else
            k_block_grad_long<T, false><<<grid, 1024, 0, st>>>(p);
        return;
    }
    const Split s = grad_split_of(p.D);
    const int threads = s.block ? s.group : 256;
#define LAUNCH(G, C, W) k_block_grad<T, G, C, W><<<grid, threads, 64 * C * threads, st>>>(p)
    SPANQR_BLOCK_SPLITS(LAUNCH)
#undef LAUNCH
}

template <typename T>
void launch_dropout(long rows, long D, const void* x, long ldx, const Dropout& drop, void* y, hipStream_t st) {
    const long pieces = (D + 7) / 8, need = (rows * pieces + DROP_PIECES - 1) / DROP_PIECES;
    k_dropout<T><<<(int)(need < 65536 ? need : 65536), 256, 0, st>>>(rows, D, (uint32_t)pieces, (const T*)x, ldx, drop, (T*)y,
                                                                             past_caches(rows, D, sizeof(T)));
}

bool known(int type) { return type == SPANQR_BF16 || type == SPANQR_FP16 || type == SPANQR_FP32; }

int check_sizes(const char* what, int type, long rows, long D, long max_D) {
    if (!known(type)) return error(SPANQR_EINVAL, "%s: unknown type", what);
    if (rows < 0 || D < 1 || D > max_D || rows > (1l << 40) / D)
        return error(SPANQR_EINVAL, "%s: rows = %ld, D = %ld (D from 1 to %ld)", what, rows, D, max_D);
    return SPANQR_OK;
}

int check_dropout(const char* what, double p, Dropout& drop, unsigned long seed, const void* seed_at, unsigned index) {
    const int below = dropped_below(p);
    if (below < 0) return error(SPANQR_EINVAL, "%s: p must be from 0 to 1 - 2^-16, got %g", what, p);
    drop = {(uint32_t)below, (float)(65536.0 / (65536.0 - below)), seed, (const uint64_t*)seed_at, index};
    return SPANQR_OK;
}

int check_block(const char* what, int type, int wtype, int act, long rows, long D) {
    const int rc = check_sizes(what, type, rows, D, MAX_D);
    if (rc != SPANQR_OK) return rc;
    if (!known(wtype)) return error(SPANQR_EINVAL, "%s: unknown type of the weights", what);
    if (act != SPANQR_GATE_LINEAR && act != SPANQR_GATE_SIGMOID && act != SPANQR_GATE_SILU)
        return error(SPANQR_EINVAL, "%s: unknown activation of the gate %d", what, act);
    return SPANQR_OK;
}

}  // namespace

extern "C" {

int spanqr_dropout(int type, long rows, long D, const void* x, long ldx, double p, unsigned long seed, const void* seed_at,
                   unsigned index, void* y, void* stream) {
    int rc = check_sizes("dropout", type, rows, D, MAX_DROP_D);
    if (rc != SPANQR_OK) return rc;
    Dropout drop;
    rc = check_dropout("dropout", p, drop, seed, seed_at, index);
    if (rc != SPANQR_OK || rows == 0) return rc;
    if (x == nullptr || y == nullptr) return error(SPANQR_EINVAL, "dropout: a missing pointer");
    if (rows > 1 && ldx < D) return error(SPANQR_EINVAL, "dropout: a row stride below D");
    hipStream_t st = (hipStream_t)stream;
    if (type == SPANQR_BF16)
        launch_dropout<bf16>(rows, D, x, ldx, drop, y, st);
    else if (type == SPANQR_FP16)
        launch_dropout<fp16>(rows, D, x, ldx, drop, y, st);
    else
        launch_dropout<float>(rows, D, x, ldx, drop, y, st);
    return launched("dropout");
}

int spanqr_block_norm(int type, int wtype, int act, long rows, long D, const void* x, long ldx, const void* residual, long ldr,
                      const void* gate, long ldg, const void* post_weight, const void* weight, float eps, float scale,
                      const float* scale_at, double p, unsigned long seed, const void* seed_at, unsigned index, void* h,
                      void* y, void* stream) {
    int rc = check_block("block_norm", type, wtype, act, rows, D);
    if (rc != SPANQR_OK) return rc;
    Dropout drop;
    rc = check_dropout("block_norm", p, drop, seed, seed_at, index);
    if (rc != SPANQR_OK || rows == 0) return rc;
    if (x == nullptr || residual == nullptr || h == nullptr || y == nullptr)
        return error(SPANQR_EINVAL, "block_norm: a missing pointer");
    if (rows > 1 && (ldx < D || ldr < D || (gate != nullptr && ldg < D)))
        return error(SPANQR_EINVAL, "block_norm: a row stride below D");
    const BlockArgs a = {rows, D, ldx, ldr, ldg, x, residual, gate, post_weight, weight, wtype, act, eps, scale, scale_at, drop,
                         h, y, past_caches(rows, D, type == SPANQR_FP32 ? 4 : 2)};
    hipStream_t st = (hipStream_t)stream;
    if (type == SPANQR_BF16)
        launch_block<bf16>(a, st);
    else if (type == SPANQR_FP16)
        launch_block<fp16>(a, st);
    else
        launch_block<float>(a, st);
    return launched("block_norm");
}

long spanqr_block_norm_backward_workspace(long rows, long D) {
    const int rc = check_sizes("block_norm_backward", SPANQR_FP32, rows, D, MAX_D);
    return rc != SPANQR_OK ? rc : 4l * grad_parts(rows, D) * (2 * D + 1);
}

int spanqr_block_norm_backward(int type, int wtype, int act, long rows, long D, const void* dy, long lddy, const void* dh,
                               long lddh, const void* x, long ldx, const void* h, long ldh, const void* gate, long ldg,
                               const void* post_weight, const void* weight, float eps, float scale, const float* scale_at,
                               double p, unsigned long seed, const void* seed_at, unsigned index, void* dx, void* dresidual,
                               void* dgate, void* dpost_weight, void* dweight, float* dscale, void* workspace,
                               long workspace_bytes, void* stream) {
    int rc = check_block("block_norm_backward", type, wtype, act, rows, D);
    if (rc != SPANQR_OK) return rc;
    Dropout drop;
    rc = check_dropout("block_norm_backward", p, drop, seed, seed_at, index);
    if (rc != SPANQR_OK) return rc;
    const bool sums = dpost_weight != nullptr || dweight != nullptr || dscale != nullptr;
    const int parts = grad_parts(rows, D);
    const long need = 4l * parts * (2 * D + 1);
    if (sums && parts > 0 && (workspace == nullptr || workspace_bytes < need))
        return error(SPANQR_EINVAL, "block_norm_backward: the workspace needs %ld bytes", need);
    hipStream_t st = (hipStream_t)stream;
    if (rows > 0) {
        if (x == nullptr || h == nullptr || dx == nullptr || dresidual == nullptr || (dgate != nullptr) != (gate != nullptr))
            return error(SPANQR_EINVAL, "block_norm_backward: a missing or needless pointer");
        if (rows > 1 && (ldx < D || ldh < D || (dy != nullptr && lddy < D) || (dh != nullptr && lddh < D) ||
                         (gate != nullptr && ldg < D)))
            return error(SPANQR_EINVAL, "block_norm_backward: a row stride below D");
        const BlockGradArgs a = {rows, D, lddy, lddh, ldx, ldh, ldg, dy, dh, x, h, gate, post_weight, weight, wtype, act, eps,
                                 scale, scale_at, drop, dx, dresidual, dgate, past_caches(rows, D, type == SPANQR_FP32 ? 4 : 2),
                                 sums ? (float*)workspace : nullptr};
        if (type == SPANQR_BF16)
            launch_grad<bf16>(a, parts, st);
        else if (type == SPANQR_FP16)
            launch_grad<fp16>(a, parts, st);
        else
            launch_grad<float>(a, parts, st);
    }
    if (sums)
        k_block_sums<<<(int)((2 * D + 16) / 16), 1024, 0, st>>>((const float*)workspace, parts, D, dpost_weight, dweight, wtype,
                                                               dscale);
    return launched("block_norm_backward");
}

}  // extern "C"
