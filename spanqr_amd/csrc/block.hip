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
// Bound by memory: each input is read once and each output written once, the row stays in registers between the two sums
// (threads and pieces as in norm.hip). Between them would be h, t, n1, dt and the mask in memory if these were operators of
// their own. Sums are fp32: per thread over at most 16 elements, then a tree in a fixed order.
#include <limits.h>

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
};

struct BlockGradArgs {
    long rows, D, lddy, lddh, ldx, ldh, ldg;
    const void *dy, *dh, *x, *h, *gate, *w1, *w2;   // dy or dh, gate and the weights may be null
    int wtype, act;
    float eps, scale;
    const float* scale_at;
    Dropout drop;
    void *dx, *dr, *dg;                          // dg null without a gate
    float* part;                                 // [gridDim.x][2 D + 1] sums over the workgroup's rows for dw1, dw2, da, or null
};

__device__ __forceinline__ float sigmoid(float g) { return 1.0f / (1.0f + expf(-g)); }

// act(g), and its slope
__device__ __forceinline__ float gate_of(int act, float g) {
    if (act == SPANQR_GATE_LINEAR) return g;
    const float s = sigmoid(g);
    return act == SPANQR_GATE_SIGMOID ? s : g * s;
}
__device__ __forceinline__ float gate_of(int act, float g, float& slope) {
    slope = 1.0f;
    if (act == SPANQR_GATE_LINEAR) return g;
    const float s = sigmoid(g);
    if (act == SPANQR_GATE_SIGMOID) {
        slope = s * (1.0f - s);
        return s;
    }
    slope = s * (1.0f + g * (1.0f - s));
    return g * s;
}

template <typename T, int GROUP, int NCH, bool WHOLE>
__global__ __launch_bounds__(Group<GROUP>::MOST) void k_block(const BlockArgs p) {
    typedef Group<GROUP> G;
    __shared__ float slot[2][2][1][16];   // both sums', by turns
    const int lane = G::lane(), size = G::size();
    const float scale = p.scale_at != nullptr ? *p.scale_at : p.scale;
    const uint64_t key = p.drop.key();
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
            if (p.gate != nullptr) kg[c] = piece<WHOLE>((const T*)p.gate + from * p.ldg, p.D, at, n);
        }
        float sum[1] = {0.0f};
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            float x[8];
            settle<WHOLE>(kx[c], on ? inside(p.D, 8l * (lane + c * size)) : 0, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[0] = fmaf(x[i], x[i], sum[0]);
        }
        G::template reduce<Sum>(sum, slot[turn][0]);
        const float s1 = rsqrtf(sum[0] / (float)p.D + p.eps);
        float h[NCH][8];
        sum[0] = 0.0f;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const long at = 8l * (lane + c * size);
            const int n = on ? inside(p.D, at) : 0;
            float x[8], w[8], f[8];
            settle<WHOLE>(kx[c], n, x);
            settle<WHOLE>(kr[c], n, h[c]);
            load_weight(p.w1, p.wtype, at, n, w);
            p.drop.factors(key, row, lane + c * size, f);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * s1 * w[i];
            if (p.gate != nullptr) {
                float g[8];
                settle<WHOLE>(kg[c], n, g);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] *= gate_of(p.act, g[i]);
            }
            // the stream is rounded as it is kept; the norm is of the rounded values
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                h[c][i] = i < n ? (float)(T)fmaf(scale, thin(x[i], f[i]), h[c][i]) : 0.0f;
                sum[0] = fmaf(h[c][i], h[c][i], sum[0]);
            }
            store8((T*)p.h + row * p.D + at, n, h[c]);
        }
        G::template reduce<Sum>(sum, slot[turn][1]);
        const float s2 = rsqrtf(sum[0] / (float)p.D + p.eps);
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const long at = 8l * (lane + c * size);
            const int n = on ? inside(p.D, at) : 0;
            float w[8];
            load_weight(p.w2, p.wtype, at, n, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[c][i] = h[c][i] * s2 * w[i];
            store8((T*)p.y + row * p.D + at, n, h[c]);
        }
    }
}

// rows longer than 16384: one workgroup a row, the row read again for each step (from the cache where it fits)
template <typename T>
__global__ __launch_bounds__(1024) void k_block_long(const BlockArgs p) {
    __shared__ float slot[16];
    const float scale = p.scale_at != nullptr ? *p.scale_at : p.scale;
    const uint64_t key = p.drop.key();
    for (long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = (const T*)p.x + row * p.ldx;
        T* h = (T*)p.h + row * p.D;
        float sum = 0.0f, v[8], w[8], f[8], g[8];
#pragma unroll 2
        for (long at = 8l * threadIdx.x; at < p.D; at += 8192) {
            settle8(fetch8(x, p.D, at), inside(p.D, at), v);
            float part = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) part = fmaf(v[i], v[i], part);
            sum += part;
        }
        sum = reduce_threads<1024, Sum>(sum, slot);
        const float s1 = rsqrtf(sum / (float)p.D + p.eps);
        sum = 0.0f;
        for (long at = 8l * threadIdx.x; at < p.D; at += 8192) {
            const int n = inside(p.D, at);
            const Pack8<T> kx = fetch8(x, p.D, at), kr = fetch8((const T*)p.residual + row * p.ldr, p.D, at);
            settle8(kx, n, v);
            load_weight(p.w1, p.wtype, at, n, w);
            p.drop.factors(key, row, at >> 3, f);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = v[i] * s1 * w[i];
            if (p.gate != nullptr) {
                settle8(fetch8((const T*)p.gate + row * p.ldg, p.D, at), n, g);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] *= gate_of(p.act, g[i]);
            }
            settle8(kr, n, g);
            float part = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[i] = i < n ? (float)(T)fmaf(scale, thin(v[i], f[i]), g[i]) : 0.0f;
                part = fmaf(v[i], v[i], part);
            }
            store8(h + at, n, v);
            sum += part;
        }
        sum = reduce_threads<1024, Sum>(sum, slot);
        const float s2 = rsqrtf(sum / (float)p.D + p.eps);
        // a thread reads back only what it wrote itself
        for (long at = 8l * threadIdx.x; at < p.D; at += 8192) {
            const int n = inside(p.D, at);
            load8(h + at, n, v);
            load_weight(p.w2, p.wtype, at, n, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = v[i] * s2 * w[i];
            store8((T*)p.y + row * p.D + at, n, v);
        }
    }
}


// The weights' gradients are sums over rows: a workgroup keeps its rows' part in registers (each thread always holds the same
// columns), adds its groups through LDS and writes one row of partial sums; k_block_sums adds those.
template <typename T, int GROUP, int NCH, bool WHOLE>
__global__ __launch_bounds__(GROUP ? 256 : 512) void k_block_grad(const BlockGradArgs p) {
    typedef Group<GROUP> G;
    __shared__ float slot[2][3][16], slot2[2][1][16];
    constexpr int ROWS = GROUP ? 256 / GROUP : 1;
    __shared__ float add[ROWS > 1 ? (ROWS - 1) * GROUP * NCH * 16 : 1];
    __shared__ float add_scale[ROWS];
    const int lane = G::lane(), group = G::index(), size = G::size();
    const float scale = p.scale_at != nullptr ? *p.scale_at : p.scale;
    const uint64_t key = p.drop.key();
    float dw1[NCH][8], dw2[NCH][8], da = 0.0f;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) dw1[c][i] = dw2[c][i] = 0.0f;
    int turn = 0;
    for (long base = (long)blockIdx.x * ROWS; base < p.rows; base += (long)gridDim.x * ROWS, turn ^= 1) {
        const long row = base + group;
        const bool on = row < p.rows;
        const long from = on ? row : base;
        Pack8<T> kx[NCH], kh[NCH], ky[NCH], kd[NCH], kg[NCH];
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const long at = 8l * (lane + c * size);
            const int n = inside(p.D, at);
            kx[c] = piece<WHOLE>((const T*)p.x + from * p.ldx, p.D, at, n);
            kh[c] = piece<WHOLE>((const T*)p.h + from * p.ldh, p.D, at, n);
#pragma unroll
            for (int i = 0; i < 8; ++i) ky[c].v[i] = kd[c].v[i] = (T)0.0f;
            if (p.dy != nullptr) ky[c] = piece<WHOLE>((const T*)p.dy + from * p.lddy, p.D, at, n);
            if (p.dh != nullptr) kd[c] = piece<WHOLE>((const T*)p.dh + from * p.lddh, p.D, at, n);
            if (p.gate != nullptr) kg[c] = piece<WHOLE>((const T*)p.gate + from * p.ldg, p.D, at, n);
        }
        float sum[3] = {0.0f, 0.0f, 0.0f};   // of x^2, h^2 and dy w2 h
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const long at = 8l * (lane + c * size);
            const int n = on ? inside(p.D, at) : 0;
            float x[8], h[8], u[8], w[8];
            settle<WHOLE>(kx[c], n, x);
            settle<WHOLE>(kh[c], n, h);
            settle<WHOLE>(ky[c], n, u);
            load_weight(p.w2, p.wtype, at, n, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sum[0] = fmaf(x[i], x[i], sum[0]);
                sum[1] = fmaf(h[i], h[i], sum[1]);
                sum[2] = fmaf(u[i] * w[i], h[i], sum[2]);
            }
        }
        G::template reduce<Sum>(sum, slot[turn]);
        // a group without a row adds zeros, also where eps is 0
        const float s1 = on ? rsqrtf(sum[0] / (float)p.D + p.eps) : 0.0f;
        const float s2 = on ? rsqrtf(sum[1] / (float)p.D + p.eps) : 0.0f;
        const float m2 = s2 * sum[2] / (float)p.D;   // the mean of dy w2 n2
        float q[NCH][8], last[1] = {0.0f};
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            again(kx[c]);   // (packed they take half the registers until here)
            again(kh[c]);
            again(ky[c]);
            const long at = 8l * (lane + c * size);
            const int n = on ? inside(p.D, at) : 0;
            float a[8], b[8], w[8], d[8], f[8];
            settle<WHOLE>(kh[c], n, a);
            settle<WHOLE>(ky[c], n, b);
            settle<WHOLE>(kd[c], n, d);
            load_weight(p.w2, p.wtype, at, n, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float n2 = a[i] * s2;
                dw2[c][i] = fmaf(b[i], n2, dw2[c][i]);
                d[i] = fmaf(s2, b[i] * w[i] - n2 * m2, d[i]);
            }
            store8((T*)p.dr + row * p.D + at, n, d);
            p.drop.factors(key, row, lane + c * size, f);
            settle<WHOLE>(kx[c], n, a);
            load_weight(p.w1, p.wtype, at, n, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                d[i] = i < n ? thin(d[i], f[i]) : 0.0f;
                a[i] *= s1;
            }
            if (p.gate != nullptr) {
                float g[8];
                settle<WHOLE>(kg[c], n, g);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float slope;
                    const float act = gate_of(p.act, g[i], slope);
                    b[i] = scale * d[i] * a[i] * w[i] * slope;
                    d[i] *= act;
                }
                store8((T*)p.dg + row * p.D + at, n, b);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                dw1[c][i] = fmaf(d[i], a[i], dw1[c][i]);
                q[c][i] = i < n ? d[i] * w[i] : 0.0f;
                last[0] = fmaf(q[c][i], a[i], last[0]);
            }
        }
        G::template reduce<Sum>(last, slot2[turn]);
        const float m1 = last[0] / (float)p.D;   // the mean of q n1
        if (lane == 0) da += last[0];
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            again(kx[c]);
            const long at = 8l * (lane + c * size);
            const int n = on ? inside(p.D, at) : 0;
            float x[8];
            settle<WHOLE>(kx[c], n, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = scale * s1 * (q[c][i] - x[i] * s1 * m1);
            store8((T*)p.dx + row * p.D + at, n, x);
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

// The gradient of rows longer than 8192, which do not stay in registers: the row is read once for each step, from L2
// behind the first one; the sums for the weights are in the partial sums' own memory, a thread's own words.
template <typename T>
__global__ __launch_bounds__(1024) void k_block_grad_long(const BlockGradArgs p) {
    __shared__ float slot[2][3][16], slot2[2][1][16];
    typedef Group<0> G;
    const float scale = p.scale_at != nullptr ? *p.scale_at : p.scale;
    const uint64_t key = p.drop.key();
    float* part = p.part == nullptr ? nullptr : p.part + blockIdx.x * (2 * p.D + 1);
    float da = 0.0f;
    int turn = 0;
    for (long row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const T* xr = (const T*)p.x + row * p.ldx;
        const T* hr = (const T*)p.h + row * p.ldh;
        const T* yr = p.dy == nullptr ? nullptr : (const T*)p.dy + row * p.lddy;
        const T* dr = p.dh == nullptr ? nullptr : (const T*)p.dh + row * p.lddh;
        const T* gr = p.gate == nullptr ? nullptr : (const T*)p.gate + row * p.ldg;
        // eight elements of a row, 0 where there is none
        auto load = [&](const T* from, long at, int n, float (&f)[8]) {
            if (from != nullptr) {
                settle8(fetch8(from, p.D, at), n, f);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = 0.0f;
            }
        };
        float sum[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll 2
        for (long at = 8l * threadIdx.x; at < p.D; at += 8192) {
            const int n = inside(p.D, at);
            float x[8], h[8], u[8], w[8], a = 0.0f, b = 0.0f, c = 0.0f;
            load(xr, at, n, x);
            load(hr, at, n, h);
            load(yr, at, n, u);
            load_weight(p.w2, p.wtype, at, n, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                a = fmaf(x[i], x[i], a);
                b = fmaf(h[i], h[i], b);
                c = fmaf(u[i] * w[i], h[i], c);
            }
            sum[0] += a;
            sum[1] += b;
            sum[2] += c;
        }
        G::template reduce<Sum>(sum, slot[turn]);
        const float s1 = rsqrtf(sum[0] / (float)p.D + p.eps), s2 = rsqrtf(sum[1] / (float)p.D + p.eps);
        const float m2 = s2 * sum[2] / (float)p.D;
        // q and n1 of a piece; in the first of two steps with everything else that the piece gives
        auto piece_of = [&](long at, int n, bool first, float (&q)[8], float (&n1)[8]) {
            float a[8], b[8], w[8], d[8], f[8], g[8];
            load(hr, at, n, a);
            load(yr, at, n, b);
            load(dr, at, n, d);
            load(gr, at, n, g);
            load(xr, at, n, n1);
            load_weight(p.w2, p.wtype, at, n, w);
            float dw2[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float n2 = a[i] * s2;
                dw2[i] = b[i] * n2;
                d[i] = fmaf(s2, b[i] * w[i] - n2 * m2, d[i]);
            }
            if (first) store8((T*)p.dr + row * p.D + at, n, d);
            p.drop.factors(key, row, at >> 3, f);
            load_weight(p.w1, p.wtype, at, n, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                d[i] = i < n ? thin(d[i], f[i]) : 0.0f;
                n1[i] *= s1;
            }
            if (gr != nullptr) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float slope;
                    const float act = gate_of(p.act, g[i], slope);
                    g[i] = scale * d[i] * n1[i] * w[i] * slope;
                    d[i] *= act;
                }
                if (first) store8((T*)p.dg + row * p.D + at, n, g);
            }
            if (first && part != nullptr) {
                float old[8];
                const bool start = row == blockIdx.x;
#pragma unroll
                for (int i = 0; i < 8; ++i) old[i] = 0.0f;
                if (!start) load8(part + at, n, old);
#pragma unroll
                for (int i = 0; i < 8; ++i) old[i] = fmaf(scale * d[i], n1[i], old[i]);
                store8(part + at, n, old);
                if (!start) load8(part + p.D + at, n, old);
#pragma unroll
                for (int i = 0; i < 8; ++i) old[i] = start ? dw2[i] : old[i] + dw2[i];
                store8(part + p.D + at, n, old);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = i < n ? d[i] * w[i] : 0.0f;
        };
        float last[1] = {0.0f}, q[8], n1[8];
        for (long at = 8l * threadIdx.x; at < p.D; at += 8192) {
            piece_of(at, inside(p.D, at), true, q, n1);
            float a = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) a = fmaf(q[i], n1[i], a);
            last[0] += a;
        }
        G::template reduce<Sum>(last, slot2[turn]);
        const float m1 = last[0] / (float)p.D;
        da += last[0];
        for (long at = 8l * threadIdx.x; at < p.D; at += 8192) {
            const int n = inside(p.D, at);
            piece_of(at, n, false, q, n1);
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = scale * s1 * (q[i] - n1[i] * m1);
            store8((T*)p.dx + row * p.D + at, n, q);
        }
    }
    if (part != nullptr && threadIdx.x == 0) part[2 * p.D] = da;
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

// Dropout alone: a workgroup takes DROP_PIECES neighbouring pieces at a time, a thread every 256th of them, so that its loads
// are under way together. pieces: of a row.
constexpr int DROP_PIECES = 1024;
template <typename T>
__global__ __launch_bounds__(256) void k_dropout(long rows, long D, uint32_t pieces, const T* x, long ldx, Dropout drop, T* y) {
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
            float v[8], f[8];
            if (D >= 8)
                settle8(k[i], n[i], v);
            else
                settle<false>(k[i], n[i], v);
            drop.factors(key, row[i], at[i] >> 3, f);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = thin(v[j], f[j]);
            store8(y + row[i] * D + at[i], n[i], v);
        }
    }
}

constexpr long LONG_ROW = 16384;   // longest row that stays in registers
constexpr long LONG_GRAD = 8192;   // and in the gradient
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

// the gradient's workgroups, and so rows of partial sums: as many as the compute units hold at once
int grad_parts(long rows, long D) {
    if (D > LONG_GRAD) return (int)(rows < 256 ? rows : 256);
    const Split s = grad_split_of(D);
    return grid_of(rows, s, !s.block || s.group <= 256 ? 1024 : 512);
}

template <typename T>
void launch_block(const BlockArgs& p, hipStream_t st) {
    if (p.D > LONG_ROW) {
        k_block_long<T><<<(int)(p.rows < 1024 ? p.rows : 1024), 1024, 0, st>>>(p);
        return;
    }
    const Split s = split_of(p.rows, p.D);
    const int grid = grid_of(p.rows, s, s.block ? 1024 : 2048);
    if (s.block && s.nch == 2)
        k_block<T, 0, 2, true><<<grid, s.group, 0, st>>>(p);
    else if (s.block)
        k_block<T, 0, 1, true><<<grid, s.group, 0, st>>>(p);
    else if (s.group == 64)
        k_block<T, 64, 1, true><<<grid, 256, 0, st>>>(p);
    else if (p.D >= 8)
        k_block<T, 16, 1, true><<<grid, 256, 0, st>>>(p);
    else
        k_block<T, 16, 1, false><<<grid, 256, 0, st>>>(p);
}

template <typename T>
void launch_grad(const BlockGradArgs& p, int grid, hipStream_t st) {
    if (p.D > LONG_GRAD) {
        k_block_grad_long<T><<<grid, 1024, 0, st>>>(p);
        return;
    }
    const Split s = grad_split_of(p.D);
    if (s.block && s.nch == 2)
        k_block_grad<T, 0, 2, true><<<grid, s.group, 0, st>>>(p);
    else if (s.block)
        k_block_grad<T, 0, 1, true><<<grid, s.group, 0, st>>>(p);
    else if (s.group == 64)
        k_block_grad<T, 64, 1, true><<<grid, 256, 0, st>>>(p);
    else if (p.D >= 8)
        k_block_grad<T, 16, 1, true><<<grid, 256, 0, st>>>(p);
    else
        k_block_grad<T, 16, 1, false><<<grid, 256, 0, st>>>(p);
}

template <typename T>
void launch_dropout(long rows, long D, const void* x, long ldx, const Dropout& drop, void* y, hipStream_t st) {
    const long pieces = (D + 7) / 8, need = (rows * pieces + DROP_PIECES - 1) / DROP_PIECES;
    k_dropout<T><<<(int)(need < 65536 ? need : 65536), 256, 0, st>>>(rows, D, (uint32_t)pieces, (const T*)x, ldx, drop, (T*)y);
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
                         h, y};
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
                                 scale, scale_at, drop, dx, dresidual, dgate, sums ? (float*)workspace : nullptr};
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
