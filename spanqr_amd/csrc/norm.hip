// norm.hip -- root-mean-square norm with the residual's addition, in the model's type or in 8 bits, and its gradient.
//
//   h = round(x + r),  s = (sum_j h_j^2 / D + eps)^(-1/2),  y_j = h_j s w_j
//   8 bits: q_j = round8(y_j M / a), scale = a / M, a = max_j |y_j|, M = 448 (fp8 e4m3) or 127 (int8); y in fp32
//   gradient: n = h s, u = dy w, dx = s (u - n sum_j(u_j n_j) / D) + dh, dw = sum over rows of dy n
//
// Both are bound by memory: one read of every input and one write of every output, with the row in registers between
// the sums and the output. A row belongs to `group` threads with NCH pieces of eight elements each: 16 lanes for up to
// 128 elements, a wavefront for up to 512 (no barriers), and then one workgroup of as many wavefronts as the row
// fills, to 1024 threads and 32768 elements; longer rows are read again for each step (k_rms_long, k_rms_grad_long).
// All sums are fp32 per thread over at most 32 elements, then a tree in a fixed order.
// 16384 x 2048 bf16 with the residual: forward 52 us (5.2 TB/s), gradient 49 and 5 for dw's parts (5.0 TB/s; part of both
// from the memory-side cache); 4096 x 5120 to 8 bits 30 us (4.9 TB/s), a copy's rate; one token of 5120 4 us.
#include "elements.h"
#include "host.h"

using namespace spanqr_dev;
using spanqr_host::error;
using spanqr_host::launched;

namespace {

struct NormArgs {
    long rows, D, ldx, ldr;
    const void *x, *residual, *weight;   // residual, weight may be null
    int wtype;                           // weight's type (SPANQR_BF16 ...)
    int quant;
    float eps;
    void *h, *y;
    float* scale;
};

struct GradArgs {
    long rows, D, lddy, ldh, lddh;
    const void *dy, *h, *weight, *dh;    // weight, dh may be null
    int wtype;
    float eps;
    void* dx;
    float* part;                         // [gridDim.x, D] sums of dy n over the block's rows, or null
};

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

__device__ __forceinline__ float quant_max(int quant) { return quant == SPANQR_QUANT_FP8 ? 448.0f : 127.0f; }

// what y is multiplied by. A row of zeros gives zeros; where M / a would overflow the largest finite factor is used.
// A NaN (of the row or of a weight) stays NaN in the scale.
__device__ __forceinline__ float quant_factor(float a, float M) {
    if (a == 0.0f) return 0.0f;
    const float f = M / a;
    return f > 3.402823466e38f ? 3.402823466e38f : f;
}

// |v| <= M by construction of the factor (up to one rounding, which round8 takes back to M)
__device__ __forceinline__ void store_quant(int quant, uint8_t* q, int n, const float (&v)[8]) {
    uint32_t lo, hi;
    if (quant == SPANQR_QUANT_FP8) {
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], 0, false);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], hi, true);
    } else {
        int k[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) k[i] = (int)rintf(v[i]);
        lo = (k[0] & 255) | (k[1] & 255) << 8 | (k[2] & 255) << 16 | (uint32_t)k[3] << 24;
        hi = (k[4] & 255) | (k[5] & 255) << 8 | (k[6] & 255) << 16 | (uint32_t)k[7] << 24;
    }
    if (n >= 8) {
        struct __attribute__((packed, aligned(1))) Two { uint32_t a, b; };
        *reinterpret_cast<Two*>(q) = Two{lo, hi};
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) q[i] = (uint8_t)((i < 4 ? lo : hi) >> 8 * (i & 3));
    }
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

template <typename T, int GROUP, int NCH, bool WHOLE>
__global__ __launch_bounds__(Group<GROUP>::MOST) void k_rms(const NormArgs p) {
    typedef Group<GROUP> G;
    __shared__ float slot[3][1][16];   // the sums' by turns, and the maximum's
    const int lane = G::lane(), size = G::size();
    float w[NCH][8];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const long at = 8l * (lane + c * size);
        load_weight(p.weight, p.wtype, at, inside(p.D, at), w[c]);
    }
    int turn = 0;
    for (long base = (long)blockIdx.x * G::rows(); base < p.rows; base += (long)gridDim.x * G::rows(), turn ^= 1) {
        const long row = base + G::index();
        const bool on = row < p.rows;   // the group's lanes all take part in the reductions
        const T* x = (const T*)p.x + (on ? row : base) * p.ldx;
        float v[NCH][8];
        Pack8<T> kx[NCH];
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const long at = 8l * (lane + c * size);
            kx[c] = piece<WHOLE>(x, p.D, at, inside(p.D, at));
        }
        if (p.residual != nullptr) {
            const T* r = (const T*)p.residual + (on ? row : base) * p.ldr;
            Pack8<T> kr[NCH];
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const long at = 8l * (lane + c * size);
                kr[c] = piece<WHOLE>(r, p.D, at, inside(p.D, at));
            }
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const long at = 8l * (lane + c * size);
                const int n = on ? inside(p.D, at) : 0;
                float u[8];
                settle<WHOLE>(kx[c], n, v[c]);
                settle<WHOLE>(kr[c], n, u);
                // the stream is rounded as it is kept; the norm is of the rounded values
#pragma unroll
                for (int i = 0; i < 8; ++i) v[c][i] = (float)(T)(v[c][i] + u[i]);
                store8((T*)p.h + row * p.D + at, n, v[c]);
            }
        } else {
#pragma unroll
            for (int c = 0; c < NCH; ++c) settle<WHOLE>(kx[c], on ? inside(p.D, 8l * (lane + c * size)) : 0, v[c]);
        }
        float sum[1] = {0.0f};
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[0] = fmaf(v[c][i], v[c][i], sum[0]);
        G::template reduce<Sum>(sum, slot[turn]);
        const float s = rsqrtf(sum[0] / (float)p.D + p.eps);
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c][i] = v[c][i] * s * w[c][i];
        if (p.quant == SPANQR_QUANT_NONE) {
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const long at = 8l * (lane + c * size);
                store8((T*)p.y + row * p.D + at, on ? inside(p.D, at) : 0, v[c]);
            }
        } else {
            // (elements past the row's end are 0, or NaN where s is: then the row is NaN anyway)
            float a[1] = {0.0f};
#pragma unroll
            for (int c = 0; c < NCH; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) a[0] = nan_max(a[0], fabsf(v[c][i]));
            G::template reduce<NanMax>(a, slot[2]);
            const float M = quant_max(p.quant), f = quant_factor(a[0], M);
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const long at = 8l * (lane + c * size);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[c][i] *= f;
                store_quant(p.quant, (uint8_t*)p.y + row * p.D + at, on ? inside(p.D, at) : 0, v[c]);
            }
            if (on && lane == 0) p.scale[row] = a[0] / M;
        }
    }
}

// rows longer than 32768: one workgroup a row, the row read again for each step (from the cache where it fits)
template <typename T>
__global__ __launch_bounds__(1024) void k_rms_long(const NormArgs p) {
    __shared__ float slot[16];
    for (long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* src = p.residual != nullptr ? (const T*)p.h + row * p.D : (const T*)p.x + row * p.ldx;
        float sum = 0.0f, v[8], w[8];
        for (long at = 8l * threadIdx.x; at < p.D; at += 8192) {
            const int n = inside(p.D, at);
            load8((const T*)p.x + row * p.ldx + at, n, v);
            if (p.residual != nullptr) {
                load8((const T*)p.residual + row * p.ldr + at, n, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = (float)(T)(v[i] + w[i]);
                store8((T*)p.h + row * p.D + at, n, v);
            }
            float part = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) part = fmaf(v[i], v[i], part);
            sum += part;
        }
        sum = reduce_threads<1024, Sum>(sum, slot);
        const float s = rsqrtf(sum / (float)p.D + p.eps);
        float a = 0.0f, f = 1.0f;
        const float M = quant_max(p.quant);
        for (int step = p.quant == SPANQR_QUANT_NONE ? 1 : 0; step < 2; ++step) {
            // a thread reads back only what it wrote itself
            for (long at = 8l * threadIdx.x; at < p.D; at += 8192) {
                const int n = inside(p.D, at);
                load8(src + at, n, v);
                load_weight(p.weight, p.wtype, at, n, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = v[i] * s * w[i];
                if (step == 0) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) a = nan_max(a, fabsf(v[i]));
                } else if (p.quant == SPANQR_QUANT_NONE) {
                    store8((T*)p.y + row * p.D + at, n, v);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] *= f;
                    store_quant(p.quant, (uint8_t*)p.y + row * p.D + at, n, v);
                }
            }
            if (step == 0) {
                a = reduce_threads<1024, NanMax>(a, slot);
                f = quant_factor(a, M);
                if (threadIdx.x == 0) p.scale[row] = a / M;
            }
        }
    }
}

// The weight's gradient is a sum over rows: a workgroup keeps its rows' part in registers (each thread always holds the
// same columns), adds its groups through LDS and writes one row of partial sums; k_rms_dw adds those.
template <typename T, int GROUP, int NCH, bool WHOLE>
__global__ __launch_bounds__(Group<GROUP>::MOST) void k_rms_grad(const GradArgs p) {
    typedef Group<GROUP> G;
    __shared__ float slot[2][2][16];
    constexpr int ROWS = GROUP ? 256 / GROUP : 1;
    __shared__ float add[ROWS > 1 ? (ROWS - 1) * GROUP * NCH * 8 : 1];
    const int lane = G::lane(), group = G::index(), size = G::size();
    float w[NCH][8], dw[NCH][8];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const long at = 8l * (lane + c * size);
        load_weight(p.weight, p.wtype, at, inside(p.D, at), w[c]);
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[c][i] = 0.0f;
    }
    int turn = 0;
    for (long base = (long)blockIdx.x * ROWS; base < p.rows; base += (long)gridDim.x * ROWS, turn ^= 1) {
        const long row = base + group;
        const bool on = row < p.rows;
        const long from = on ? row : base;
        Pack8<T> kh[NCH], ku[NCH], kd[NCH];
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const long at = 8l * (lane + c * size);
            const int n = inside(p.D, at);
            kh[c] = piece<WHOLE>((const T*)p.h + from * p.ldh, p.D, at, n);
            ku[c] = piece<WHOLE>((const T*)p.dy + from * p.lddy, p.D, at, n);
        }
        if (p.dh != nullptr) {
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const long at = 8l * (lane + c * size);
                kd[c] = piece<WHOLE>((const T*)p.dh + from * p.lddh, p.D, at, inside(p.D, at));
            }
        } else {
#pragma unroll
            for (int c = 0; c < NCH; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) kd[c].v[i] = (T)0.0f;
        }
        float sum[2] = {0.0f, 0.0f};   // of h^2, and of u h
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            float h[8], u[8];
            const int n = on ? inside(p.D, 8l * (lane + c * size)) : 0;
            settle<WHOLE>(kh[c], n, h);
            settle<WHOLE>(ku[c], n, u);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sum[0] = fmaf(h[i], h[i], sum[0]);
                sum[1] = fmaf(u[i] * w[c][i], h[i], sum[1]);
            }
        }
        G::template reduce<Sum>(sum, slot[turn]);
        // a group without a row adds zeros, also where eps is 0
        const float s = on ? rsqrtf(sum[0] / (float)p.D + p.eps) : 0.0f;
        const float m = s * sum[1] / (float)p.D;   // the mean of u n
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            again(kh[c]);   // (packed they take half the registers until here)
            again(ku[c]);
            const long at = 8l * (lane + c * size);
            const int n = on ? inside(p.D, at) : 0;
            float h[8], u[8], d[8];
            settle<WHOLE>(kh[c], n, h);
            settle<WHOLE>(ku[c], n, u);
            settle<WHOLE>(kd[c], n, d);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float nrm = h[i] * s;
                dw[c][i] = fmaf(u[i], nrm, dw[c][i]);
                d[i] = fmaf(s, u[i] * w[c][i] - nrm * m, d[i]);
            }
            store8((T*)p.dx + row * p.D + at, n, d);
        }
    }
    if (p.part == nullptr) return;
    if constexpr (ROWS > 1) {
        if (group > 0) {
#pragma unroll
            for (int c = 0; c < NCH; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) add[((group - 1) * NCH * 8 + c * 8 + i) * GROUP + lane] = dw[c][i];
        }
        __syncthreads();
        if (group > 0) return;
        for (int g = 0; g < ROWS - 1; ++g)
#pragma unroll
            for (int c = 0; c < NCH; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) dw[c][i] += add[(g * NCH * 8 + c * 8 + i) * GROUP + lane];
    }
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const long at = 8l * (lane + c * size);
        store8(p.part + blockIdx.x * p.D + at, inside(p.D, at), dw[c]);
    }
}

// The gradient of rows longer than 16384, whose sums for dw would not stay in registers beside the row: the row is
// read twice (from L2 the second time), and the sums are in LDS (up to 32768 columns), or in the partial sums' own memory.
template <typename T, bool IN_LDS>
__global__ __launch_bounds__(1024) void k_rms_grad_long(const GradArgs p) {
    __shared__ float slot[2][2][16];
    __shared__ float add[IN_LDS ? 32768 : 1];
    typedef Group<0> G;
    const int t = threadIdx.x;
    if constexpr (IN_LDS) {
        for (int i = t; i < 32768; i += 1024) add[i] = 0.0f;   // (a thread's own words)
    }
    int turn = 0;
    for (long row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const T* hr = (const T*)p.h + row * p.ldh;
        const T* ur = (const T*)p.dy + row * p.lddy;
        float h[8], u[8], w[8], d[8];
        float sum[2] = {0.0f, 0.0f};
#pragma unroll 2
        for (long at = 8l * t; at < p.D; at += 8192) {
            const int n = inside(p.D, at);
            const Pack8<T> kh = fetch8(hr, p.D, at), ku = fetch8(ur, p.D, at);
            load_weight(p.weight, p.wtype, at, n, w);
            settle8(kh, n, h);
            settle8(ku, n, u);
            float a = 0.0f, b = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                a = fmaf(h[i], h[i], a);
                b = fmaf(u[i] * w[i], h[i], b);
            }
            sum[0] += a;
            sum[1] += b;
        }
        G::template reduce<Sum>(sum, slot[turn]);
        const float s = rsqrtf(sum[0] / (float)p.D + p.eps);
        const float m = s * sum[1] / (float)p.D;
        float* mine = add + t;
#pragma unroll 2
        for (long at = 8l * t; at < p.D; at += 8192, mine += 8192) {
            const int n = inside(p.D, at);
            const Pack8<T> kh = fetch8(hr, p.D, at), ku = fetch8(ur, p.D, at);
            if (p.dh != nullptr) {
                settle8(fetch8((const T*)p.dh + row * p.lddh, p.D, at), n, d);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] = 0.0f;
            }
            load_weight(p.weight, p.wtype, at, n, w);
            settle8(kh, n, h);
            settle8(ku, n, u);
            float dw[8];
            float* part = p.part == nullptr ? nullptr : p.part + blockIdx.x * p.D + at;
            if (!IN_LDS && part != nullptr && row != blockIdx.x) {
                load8(part, n, dw);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) dw[i] = IN_LDS ? mine[1024 * i] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float nrm = h[i] * s;
                dw[i] = fmaf(u[i], nrm, dw[i]);
                d[i] = fmaf(s, u[i] * w[i] - nrm * m, d[i]);
            }
            store8((T*)p.dx + row * p.D + at, n, d);
            if constexpr (IN_LDS) {
#pragma unroll
                for (int i = 0; i < 8; ++i) mine[1024 * i] = dw[i];
            } else if (part != nullptr) {
                store8(part, n, dw);
            }
        }
    }
    if (IN_LDS && p.part != nullptr) {
        const float* mine = add + t;
        for (long at = 8l * t; at < p.D; at += 8192, mine += 8192) {
            float dw[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) dw[i] = mine[1024 * i];
            store8(p.part + blockIdx.x * p.D + at, inside(p.D, at), dw);
        }
    }
}

// dw[d] = sum of part[0..parts)[d]: 16 columns a workgroup, 64 threads a column, added in a fixed order
__global__ __launch_bounds__(1024) void k_rms_dw(const float* part, int parts, long D, void* dw, int wtype) {
    __shared__ float add[64][17];
    const int col = threadIdx.x & 15, at = threadIdx.x >> 4;
    long d = 16l * blockIdx.x + col;
    float sum = 0.0f;
    if (d < D) {
#pragma unroll 8
        for (int i = at; i < parts; i += 64) sum += part[i * D + d];
    }
    add[at][col] = sum;
    __syncthreads();
    // a wavefront a column
    d = 16l * blockIdx.x + (threadIdx.x >> 6);
    sum = reduce_lanes<64, Sum>(add[threadIdx.x & 63][threadIdx.x >> 6]);
    if ((threadIdx.x & 63) != 0 || d >= D) return;
    if (wtype == SPANQR_BF16)
        ((bf16*)dw)[d] = (bf16)sum;
    else if (wtype == SPANQR_FP16)
        ((fp16*)dw)[d] = (fp16)sum;
    else
        ((float*)dw)[d] = sum;
}

constexpr long LONG_ROW = 32768;    // longest row that stays in registers
constexpr long LONG_GRAD = 16384;   // and in the gradient
constexpr long MAX_D = 1l << 24;

// Threads of a row and pieces a thread. Measured, forward / backward in us: 16384 x 2048 bf16 as 256 threads of one
// piece 51 / 50, as 128 of two 53 / 53, as a wavefront of four 60 / 55; 4096 x 5120 with 8 bits as 640 of one 40, as 320
// of two 31, as 192 of four 35. One token of 5120 as 640 of one 3.8, as 256 of four 6.7.
struct Split {
    int group, nch;   // group 16 or 64: lanes of a wavefront; else (64 and `block`) a workgroup
    bool block;
};
Split split_of(long rows, long D) {
    const long pieces = (D + 7) / 8;
    if (D <= 128) return {16, 1, false};
    if (D <= 512) return {64, 1, false};
    const int nch = D <= 2048 || (rows <= 512 && D <= 8192) ? 1 : D <= 16384 ? 2 : 4;
    return {(int)(((pieces + nch - 1) / nch + 63) / 64 * 64), nch, true};
}

// workgroups for `rows` rows, each of about as many rows as the others, `most` at most
int grid_of(long rows, const Split& s, int most) {
    const int per = s.block ? 1 : 256 / s.group;
    const long need = (rows + per - 1) / per, turns = (need + most - 1) / most;
    return turns < 1 ? 0 : (int)((need + turns - 1) / turns);
}

// The gradient's workgroups, and so rows of partial sums: as many as the compute units hold at once, since each of them ends
// with a row of sums that is written and read again. The gradient and dw, in us, with 1024 / 512 / 256: rows of 4000 (256
// threads) 49 + 7 / 54 + 6 / 84 + 4, 4096 of 5120 (320) 46 + 9 / 34 + 6 / 49 + 4, 2000 of 12000 (768) 59 + 18 / 51 + 13 / 46 + 7.
int grad_parts(long rows, long D) {
    if (D > LONG_GRAD) return (int)(rows < 256 ? rows : 256);
    const Split s = split_of(rows, D);
    return grid_of(rows, s, !s.block || s.group <= 256 ? 1024 : s.group <= 512 ? 512 : 256);
}

#define SPANQR_SPLITS(LAUNCH)                                       \
    if (s.block) {                                                  \
        if (s.nch == 1) LAUNCH(0, 1, true, s.group);                \
        else if (s.nch == 2) LAUNCH(0, 2, true, s.group);           \
        else LAUNCH(0, 4, true, s.group);                           \
    } else if (s.group == 16) {                                     \
        if (p.D >= 8) LAUNCH(16, 1, true, 256);                     \
        else LAUNCH(16, 1, false, 256);                             \
    } else {                                                        \
        LAUNCH(64, 1, true, 256);                                   \
    }

template <typename T>
void launch_norm(const NormArgs& p, hipStream_t st) {
    if (p.D > LONG_ROW) {
        k_rms_long<T><<<(int)(p.rows < 1024 ? p.rows : 1024), 1024, 0, st>>>(p);
        return;
    }
    const Split s = split_of(p.rows, p.D);
    const int grid = grid_of(p.rows, s, s.block ? 1024 : 2048);
#define LAUNCH(G, C, W, N) k_rms<T, G, C, W><<<grid, N, 0, st>>>(p)
    SPANQR_SPLITS(LAUNCH)
#undef LAUNCH
}

template <typename T>
void launch_grad(const GradArgs& p, int grid, hipStream_t st) {
    if (p.D > LONG_GRAD) {
        if (p.D <= 32768)
            k_rms_grad_long<T, true><<<grid, 1024, 0, st>>>(p);
        else
            k_rms_grad_long<T, false><<<grid, 1024, 0, st>>>(p);
        return;
    }
    const Split s = split_of(p.rows, p.D);
#define LAUNCH(G, C, W, N) k_rms_grad<T, G, C == 4 ? 2 : C, W><<<grid, N, 0, st>>>(p)   // (four pieces: rows above 16384)
    SPANQR_SPLITS(LAUNCH)
#undef LAUNCH
}

bool known(int type) { return type == SPANQR_BF16 || type == SPANQR_FP16 || type == SPANQR_FP32; }

int check_sizes(const char* what, int type, int wtype, long rows, long D) {
    if (!known(type) || !known(wtype)) return error(SPANQR_EINVAL, "%s: unknown type", what);
    if (rows < 0 || D < 1 || D > MAX_D || rows > (1l << 40) / D)
        return error(SPANQR_EINVAL, "%s: rows = %ld, D = %ld (D from 1 to %ld)", what, rows, D, MAX_D);
    return SPANQR_OK;
}

}  // namespace

extern "C" {

int spanqr_rms_norm(int type, int wtype, int quant, long rows, long D, const void* x, long ldx, const void* residual,
                    long ldr, const void* weight, float eps, void* h, void* y, float* scale, void* stream) {
    const int rc = check_sizes("rms_norm", type, wtype, rows, D);
    if (rc != SPANQR_OK) return rc;
    if (quant != SPANQR_QUANT_NONE && quant != SPANQR_QUANT_FP8 && quant != SPANQR_QUANT_INT8)
        return error(SPANQR_EINVAL, "rms_norm: unknown quant %d", quant);
    if (rows == 0) return SPANQR_OK;
    if (x == nullptr || y == nullptr || (residual != nullptr) != (h != nullptr) ||
        (quant != SPANQR_QUANT_NONE) != (scale != nullptr))
        return error(SPANQR_EINVAL, "rms_norm: a missing or needless pointer");
    if (rows > 1 && (ldx < D || (residual != nullptr && ldr < D)))
        return error(SPANQR_EINVAL, "rms_norm: a row stride below D");
    const NormArgs p = {rows, D, ldx, ldr, x, residual, weight, wtype, quant, eps, h, y, scale};
    hipStream_t st = (hipStream_t)stream;
    if (type == SPANQR_BF16)
        launch_norm<bf16>(p, st);
    else if (type == SPANQR_FP16)
        launch_norm<fp16>(p, st);
    else
        launch_norm<float>(p, st);
    return launched("rms_norm");
}

long spanqr_rms_norm_backward_workspace(long rows, long D) {
    if (rows < 0 || D < 1 || D > MAX_D) return error(SPANQR_EINVAL, "rms_norm_backward: rows = %ld, D = %ld", rows, D);
    return 4l * grad_parts(rows, D) * D;
}

int spanqr_rms_norm_backward(int type, int wtype, long rows, long D, const void* dy, long lddy, const void* h, long ldh,
                             const void* weight, const void* dh, long lddh, float eps, void* dx, void* dw,
                             void* workspace, long workspace_bytes, void* stream) {
    const int rc = check_sizes("rms_norm_backward", type, wtype, rows, D);
    if (rc != SPANQR_OK) return rc;
    const int parts = grad_parts(rows, D);
    if (dw != nullptr && parts > 0 && (workspace == nullptr || workspace_bytes < 4l * parts * D))
        return error(SPANQR_EINVAL, "rms_norm_backward: the workspace needs %ld bytes", 4l * parts * D);
    hipStream_t st = (hipStream_t)stream;
    if (rows > 0) {
        if (dy == nullptr || h == nullptr || dx == nullptr)
            return error(SPANQR_EINVAL, "rms_norm_backward: a missing pointer");
        if (rows > 1 && (lddy < D || ldh < D || (dh != nullptr && lddh < D)))
            return error(SPANQR_EINVAL, "rms_norm_backward: a row stride below D");
        const GradArgs p = {rows, D, lddy, ldh, lddh, dy, h, weight, dh, wtype, eps, dx,
                            dw == nullptr ? nullptr : (float*)workspace};
        if (type == SPANQR_BF16)
            launch_grad<bf16>(p, parts, st);
        else if (type == SPANQR_FP16)
            launch_grad<fp16>(p, parts, st);
        else
            launch_grad<float>(p, parts, st);
    }
    if (dw != nullptr)
        k_rms_dw<<<(int)((D + 15) / 16), 1024, 0, st>>>((const float*)workspace, parts, D, dw, wtype);
    return launched("rms_norm_backward");
}

}  // extern "C"
